"""The oracle's laws of the paged cache and of attention over it, by hand-worked cases and identities,
and the refusals of the C entries that come before any device call. No GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from cozyq import _lib, kv_cache
from oracle import cache as law

INVALID = 1


def test_plan_by_hand():
    """Pages of 4: request 0 holds 3 and brings 2 (the rest of its page and one of a new one), request 1
    begins, request 2 brings none, request 3 finds the list empty after its first page."""
    p = law.plan([[7, -1, -1], [-1, -1, -1], [5, -1, -1], [-1, -1, -1]], [4, 6, 9], 3, [3, 0, 2, 0], [2, 1, 0, 5], 10, 4)
    assert p["table"] == [[7, 9, -1], [6, -1, -1], [5, -1, -1], [4, -1, -1]]
    assert p["starts"] == [0, 2, 3, 3, 8] and p["lengths"] == [5, 1, 2, 5]
    assert p["positions"] == [3, 4, 0, 0, 1, 2, 3, 4, 0, 0]
    assert p["requests"] == [0, 0, 1, 3, 3, 3, 3, 3, -1, -1]
    assert p["slots"] == [31, 36, 24, 16, 17, 18, 19, -1, -1, -1]
    assert p["runs"][:5] == [[0, 1, 7, 3], [1, 1, 9, 0], [2, 1, 6, 0], [3, 4, 4, 0], [7, 1, -1, 0]]
    assert p["spare"] == [0, 1] and len(p["runs"]) == 10


def test_append_rounds_again_when_the_scale_grows():
    """One head of width 2, pages of 4, int8: 127 units of 1/127, then a token twice as large."""
    codes, scale = torch.zeros(1, 1, 4, 2), torch.full((1, 1), 9.0)
    law.append(codes, scale, torch.tensor([[[1.0, -0.5]]]), [[0, 1, 0, 0]], torch.int8)
    assert codes[0, 0, 0].tolist() == [127.0, -64.0] and scale.item() == pytest.approx(1 / 127)
    assert codes[0, 0, 1:].abs().sum() == 0
    law.append(codes, scale, torch.tensor([[[0.25, 2.0]]]), [[0, 1, 0, 1]], torch.int8)
    assert codes[0, 0, :2].tolist() == [[64.0, -32.0], [16.0, 127.0]] and scale.item() == pytest.approx(2 / 127)
    law.append(codes, scale, torch.tensor([[[math.nan, 1.0]]]), [[0, 1, 0, 2]], torch.int8)
    assert scale.isnan().all() and codes.isfinite().all()


def test_attend_of_equal_keys_is_the_mean_and_of_one_token_its_value():
    k = torch.ones(2, 1, 16, 64)
    v = torch.randn(2, 1, 16, 64, generator=torch.Generator().manual_seed(1))
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(2))
    out, _ = law.attend(q, k, v, [[1, 0]], [0, 2], [20], 16)
    mean = torch.cat((v[1, 0], v[0, 0, :4])).double().mean(0)
    assert torch.allclose(out[1, 0], mean, atol=1e-12)
    out, _ = law.attend(q, k, v, [[1, 0]], [0, 2], [20], 16, window=1)
    assert torch.allclose(out[0, 1], v[0, 0, 2].double(), atol=1e-12)
    out, _ = law.attend(q, k, v, [[-1, -1]], [0, 2], [20], 16)
    assert out.abs().sum() == 0


def test_norm_rope_turns_by_the_angle_and_keeps_the_norm():
    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(3))
    angle = torch.rand(3, 16, generator=torch.Generator().manual_seed(4))
    for pairs in (False, True):
        y, _ = law.norm_rope(x, None, angle.cos(), angle.sin(), None, None, pairs)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1), rtol=1e-6)
        assert torch.equal(y[..., 32:], x[..., 32:].double())
        back, _ = law.norm_rope(y, None, angle.cos(), -angle.sin(), None, None, pairs)
        assert torch.allclose(back, x.double(), atol=1e-6)


def _buffer():
    buf = ctypes.create_string_buffer(4096 + 16)
    return buf, ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16


def test_entries_refuse_bad_arguments_before_the_device():
    lib = _lib.load()
    keep, p = _buffer()
    assert lib.cozyq_cache_most_requests() == 4000
    assert lib.cozyq_cache_runs(10, 4, 4) == -1 and lib.cozyq_cache_runs(10, 4, 48) == -1
    assert lib.cozyq_cache_runs(100, 2, 16) == 10 and lib.cozyq_cache_runs(3, 2, 16) == 3
    assert lib.cozyq_cache_runs(-1, 2, 16) == -1 and lib.cozyq_cache_runs(1, 4001, 16) == -1

    def rope(q=p, tokens=1, q_heads=1, k_heads=1, width=64, stride=64, cos=p, rows=4, rotated=64, positions=None, out=p):
        return lib.cozyq_head_norm_rope(0, q, p, 0, tokens, q_heads, k_heads, width, stride, stride, stride, stride, 1,
                                        None, None, 0, 1e-6, cos, p, rows, rotated, 0, positions, out, p, None)  # fmt: skip

    assert rope(tokens=0) == 0 and rope(q_heads=0, k_heads=0) == 0
    for bad in (dict(width=72), dict(width=272), dict(width=0), dict(rotated=80), dict(rotated=24), dict(stride=60),
                dict(q=p + 8), dict(q=None), dict(out=None), dict(cos=None), dict(rows=0), dict(tokens=5), dict(tokens=-1)):  # fmt: skip
        assert rope(**bad) == INVALID, bad

    def plan(table=p, requests=1, width=2, free=p, count=1, tokens=1, page=16, runs=p):
        return lib.cozyq_cache_plan(0, table, requests, width, free, count, p, p, p, tokens, page, p, p, p, p, p, runs, p, None)

    for bad in (dict(table=None), dict(requests=0), dict(requests=4001), dict(width=0), dict(free=None), dict(page=24),
                dict(page=8), dict(tokens=-1), dict(runs=None), dict(runs=p + 4), dict(count=-1)):  # fmt: skip
        assert plan(**bad) == INVALID, bad

    def append(k=p, tokens=1, step=64, codes=p, pages=1, heads=1, page=16, width=64, runs=p, most=1):
        return lib.cozyq_cache_append(0, 0, k, p, 0, tokens, step, step, step, step, codes, p, p, p, pages, heads, page,
                                      width, runs, most, None)  # fmt: skip

    assert append(tokens=0) == 0 and append(most=0) == 0
    for bad in (dict(k=None), dict(k=p + 2), dict(step=4), dict(codes=p + 8), dict(pages=0), dict(heads=0), dict(page=12),
                dict(width=96), dict(runs=None), dict(most=-1)):  # fmt: skip
        assert append(**bad) == INVALID, bad

    def read(codes=p, count=1, width=64, out=p, numbers=p):
        return lib.cozyq_cache_read(0, 1, codes, p, p, p, 1, 1, 16, width, numbers, count, out, p, 0, None)

    assert read(count=0) == 0
    for bad in (dict(codes=None), dict(count=-1), dict(width=32), dict(out=p + 8), dict(numbers=None)):
        assert read(**bad) == INVALID, bad

    def attend(q=p, tokens=1, q_heads=2, step=64, heads=1, page=16, width=64, table=p, requests=1, columns=1, most=1,
               causal=1, window=0, out=p):  # fmt: skip
        return lib.cozyq_cache_attend(0, 0, q, 0, tokens, q_heads, step, step, p, p, p, p, 1, heads, page, width, table,
                                      requests, columns, p, p, most, 1.0, causal, window, out, p, None)  # fmt: skip

    assert attend(tokens=0) == 0
    for bad in (dict(q=None), dict(q=p + 2), dict(q_heads=3, heads=2), dict(q_heads=65), dict(step=12), dict(page=20),
                dict(width=80), dict(table=None), dict(requests=0), dict(requests=4001), dict(columns=0), dict(most=-1),
                dict(window=-1), dict(causal=0, window=4), dict(out=None), dict(out=p + 4), dict(tokens=-1)):  # fmt: skip
        assert attend(**bad) == INVALID, bad
    assert lib.cozyq_cache_attend_workspace_bytes(1, 3, 1, 2, 16, 64, 4, 1, 0) == -1
    assert lib.cozyq_cache_attend_workspace_bytes(1, 2, 1, 2, 16, 64, 4, 1, 0) >= 0
    del keep


def test_cpu_tensors_and_wrong_types_are_refused():
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    from cozyq import heads

    with pytest.raises(ValueError, match="gfx950"):
        heads.norm_rope(torch, x, x, None, None, None, None)
    with pytest.raises(ValueError, match="gfx950"):
        kv_cache.plan(torch, torch.zeros(1, 1, dtype=torch.int32), x, x, x, x, tokens=1, page=16)
    cache = kv_cache.empty(torch, 2, 1, 64, page=32, device="cpu")
    assert cache.page == 32 and cache.v.shape == (2, 1, 64, 32) and cache.k.dtype is torch.int8
    with pytest.raises(ValueError, match="gfx950"):
        cache.attend(torch, x, None)
    for bad in (dict(page=24), dict(width=80), dict(dtype=torch.bfloat16), dict(pages=0)):
        args = dict(pages=2, heads=1, width=64, page=32, dtype=torch.int8) | bad
        with pytest.raises(ValueError):
            kv_cache.empty(torch, args["pages"], args["heads"], args["width"], page=args["page"], dtype=args["dtype"], device="cpu")
