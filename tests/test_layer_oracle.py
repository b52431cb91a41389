"""The oracle's laws of the residual norm, of positions on several axes and of attention to an encoder's states, by
hand-worked cases and identities, and the refusals of the C entries that come before any device call. No GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from cozyq import _lib, norms
from oracle import cache, laws, layer

INVALID = 1


def test_the_rotation_is_the_int8_linears():
    x = torch.randn(3, 512, generator=torch.Generator().manual_seed(1))
    h = layer.hadamard256()
    assert torch.allclose(h @ h.T, torch.eye(256, dtype=torch.float64), atol=1e-12)
    want = laws.int8_weight_rotated(x, 256)
    turned = (x.double().view(-1, 256) @ h).view(3, 512)
    codes = (turned / (turned.abs().amax(-1, keepdim=True) / 127)).round()
    assert (codes - want[0].double()).abs().max() <= 1 and (codes == want[0].double()).double().mean() > 0.999


def test_add_rms_by_hand():
    """3 + 1 and 4 - 1: a sum of (4, 3) and fourteen zeros has the mean square 25 / 16."""
    x, r = torch.zeros(1, 16).bfloat16(), torch.zeros(1, 16).bfloat16()
    x[0, :2], r[0, :2] = torch.tensor([3.0, 4.0]), torch.tensor([1.0, -1.0])
    total, n, scale, _ = layer.add_rms(x, r, torch.full((16,), 2.0), torch.float8_e4m3fn, 1e-30)
    assert total[0, :2].tolist() == [4.0, 3.0]
    assert n[0, :3].tolist() == pytest.approx([6.4, 4.8, 0.0]) and scale.item() == pytest.approx(6.4 / 448)


def test_axes_of_pairs():
    assert layer.axis_of_pairs((2, 1, 3), False) == [0, 0, 1, 2, 2, 2]
    assert layer.axis_of_pairs((4, 2, 2), True) == [0, 1, 2, 0, 1, 2, 0, 0]
    cos = torch.arange(12.0).view(6, 2)
    c, _ = layer.tables(cos, cos, torch.tensor([[1, 9], [2, -1]]), (1, 1), False)
    assert c.tolist() == [[2.0, 5.0], [10.0, 1.0]]


def test_axes_that_agree_are_one_axis():
    gen = torch.Generator().manual_seed(2)
    x, angle = torch.randn(4, 2, 32, generator=gen), torch.rand(9, 8, generator=gen)
    at = torch.tensor([3, 0, 8, 5])
    one, _ = cache.norm_rope(x, None, angle.cos(), angle.sin(), at, None, False)
    c, s = layer.tables(angle.cos(), angle.sin(), torch.stack((at, at, at)), (3, 3, 2), True)
    many, _ = cache.norm_rope(x, None, c, s, None, None, False)
    assert torch.equal(one, many)


def test_cross_of_equal_keys_is_the_mean_and_of_one_state_its_value():
    gen = torch.Generator().manual_seed(3)
    q, v = torch.randn(5, 2, 16, generator=gen), torch.randn(3, 6, 1, 16, generator=gen)
    k = torch.ones(3, 6, 1, 16)
    mask = torch.ones(3, 6, dtype=torch.bool)
    mask[0, 1:5] = False
    mask[2] = False
    out, _ = layer.cross(q, k, v, [0, 2, 3, 4], [6, 1, 6], mask)
    assert torch.allclose(out[1, 0], v[0, [0, 5], 0].double().mean(0), atol=1e-12)
    assert torch.allclose(out[2, 1], v[1, 0, 0].double(), atol=1e-12)
    assert out[3].abs().sum() == 0 and out[4].abs().sum() == 0


def _buffer():
    buf = ctypes.create_string_buffer(4096 + 16)
    return buf, ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16


def test_add_rms_entry_refuses_bad_arguments_before_the_device():
    lib = _lib.load()
    keep, p = _buffer()

    def call(fp8=0, x=p, residual=p, gain=None, eps=1e-6, total=p, codes=p, scales=p, rows=1, width=256):
        return lib.cozyq_add_rms(0, fp8, x, residual, 0, gain, 0, eps, total, codes, scales, rows, width, None)

    for bad in (dict(x=None), dict(x=p + 2), dict(residual=p + 2), dict(total=None), dict(total=p + 8), dict(codes=None),
                dict(codes=p + 4), dict(scales=None), dict(gain=p + 4), dict(eps=0.0), dict(eps=-1.0), dict(eps=math.nan),
                dict(rows=-1), dict(rows=2**30 + 1), dict(width=0), dict(width=128), dict(width=32768 + 256),
                dict(fp8=1, width=24)):  # fmt: skip
        assert call(**bad) == INVALID, bad
    assert call(rows=0) == 0


def test_rope_axes_entry_refuses_bad_arguments_before_the_device():
    lib = _lib.load()
    keep, p = _buffer()

    def call(axes=3, sections=(8, 12, 12), cycled=0, positions=p, rotated=64):
        shares = None if sections is None else (ctypes.c_int * len(sections))(*sections)
        return lib.cozyq_head_norm_rope_axes(0, p, p, 0, 1, 1, 1, 64, 64, 64, 64, 64, 1, None, None, 0, 1e-6, p, p, 4,
                                             rotated, 0, positions, axes, shares, cycled, p, p, None)  # fmt: skip

    for bad in (dict(axes=0), dict(axes=5, sections=(8, 6, 6, 6, 6)), dict(sections=None), dict(positions=None),
                dict(sections=(8, 12, 11)), dict(sections=(8, 12, 13)), dict(sections=(8, -4, 28)), dict(rotated=0),
                dict(sections=(2, 15, 15), cycled=1), dict(sections=(2**30, 2**30, 2**30))):  # fmt: skip
        assert call(**bad) == INVALID, bad


def test_operators_refuse_tensors_off_the_gpu_and_unknown_operands():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        norms.add_rms(torch, x, x, None)


def test_cross_entry_refuses_bad_arguments_before_the_device():
    lib = _lib.load()
    keep, p = _buffer()

    def call(q=p, tokens=4, q_heads=4, q_token=256, k=p, v=p, requests=2, states=8, kv_heads=2, width=64, k_state=128, v_state=128,
             starts=p, most=0, out=p, k_head=64):  # fmt: skip
        return lib.cozyq_cross_attend(0, q, 0, tokens, q_heads, q_token, 64, k, v, requests, states, kv_heads, width, 1024, k_state,
                                      k_head, 1024, v_state, 64, starts, p, None, 0, most, 0.1, out, None, None)  # fmt: skip

    for bad in (dict(q=None), dict(q=p + 2), dict(k=None), dict(v=p + 8), dict(out=None), dict(out=p + 4), dict(tokens=-1), dict(tokens=2**30 + 1),
                dict(tokens=2**29, q_heads=8), dict(q_heads=3), dict(q_heads=0), dict(kv_heads=0), dict(requests=0), dict(requests=65536),
                dict(states=-1), dict(width=0), dict(width=12), dict(width=264), dict(q_token=100), dict(k_state=100), dict(k_head=4),
                dict(k_state=1 << 23), dict(v_state=-8), dict(most=-1), dict(starts=None, tokens=5)):  # fmt: skip
        assert call(**bad) == INVALID, bad
    assert call(tokens=0) == 0
    size = lib.cozyq_cross_attend_workspace_bytes
    assert size(4, 4, 0, 8, 2, 64, 0) == -1 and size(4, 4, 2, 8, 2, 64, -1) == -1 and size(4, 4, 2, 8, 2, 64, 0) == 0
