"""Attention to an encoder's states (`cozyq.attention.cross`) where every state counts, at the ends of its types and at
scores far from zero, against counts and `oracle/layer.py`; bars as in test_gpu_cross.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cross import BF16, FP16, check, counts, inputs
from test_gpu_kv_cache import DEV, UNIT, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attention():
    from cozyq import attention

    return attention


# One row and a few, two tiles of few rows, part of a tile of many, more than one.
ROWS = [[1, 2], [20], [60, 1], [130, 1], [300]]


@pytest.mark.parametrize("width,dtype", [(64, FP16), (128, FP16), (256, BF16), (256, FP16)])
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_cross_every_state_counts_once(attention, rows, width, dtype):
    """Keys of zeros and values of one channel each, state t's the channel t % D: the result is how many of a request's n
    states have the channel, over n. Weights (2^6 or 2^-14) and their sums (below 2^15 states) are exact, so that the
    quotient's two roundings in float32 and the output's one are all there is: u + 2^-22. A state lost or taken twice
    moves its channel's count of 16385 states by one in 64, 128 or 256 (D 256, 128, 64), that is by eight times u or more
    in fp16 and by four times in bf16, and fewer states' by more."""
    for states in (1, 31, 32, 33, 64, 65, 127, 255, 257, 767, 769, 1025, 4096, 4097, 16385):
        requests = len(rows)
        q, _, _ = inputs(sum(rows), requests, 1, 2, 1, width, dtype, states)
        k = torch.zeros(requests, states, 1, width, dtype=dtype, device=DEV)
        t = torch.arange(states, device=DEV)
        channel = torch.nn.functional.one_hot(t % width, width)
        v = channel.to(dtype)[None, :, None].expand(requests, -1, -1, -1)
        lengths = [states, max(1, states - 2)][:requests]
        gen = torch.Generator(DEV).manual_seed(states)
        mask = torch.rand(requests, states, generator=gen, device=DEV) < 0.8
        mask[:, ::97] = True
        for shown in (None, mask):
            got = attention.cross(torch, q, k, v, starts=counts(rows), lengths=ints(lengths), mask=shown, most=max(rows))
            for r, n in enumerate(lengths):
                seen = t < n if shown is None else (t < n) & shown[r]
                want = channel[seen].sum(0).double() / int(seen.sum())
                mine = got[sum(rows[:r]) : sum(rows[: r + 1])].double()
                assert ((mine - want).abs() <= (UNIT[dtype] + 2.0**-22) * want).all(), (states, r)


@pytest.mark.parametrize("states", [40, 450, 5000])
@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("power", [126, 60, -100, -120, -126])
def test_cross_values_of_any_size(attention, rows, states, power):
    """bf16 values near the type's ends: their weighted means are as large, whatever their sums would be. Scores grow
    along the states, so that the largest is met late. Sums of the smallest are in steps of 2^-149, half of which every
    16 states (a matrix instruction) may cost over weights of 2^-14 and more: 2^-131 of the mean for 450, below the bars'
    2^-130, and for 5000 2^-128, below their 2^-127 at 2^-120."""
    if power == -126 and states > 450:
        pytest.skip("past what float32's smallest steps allow")
    q, k, v = inputs(sum(rows), len(rows), states, 4, 2, 64, BF16, states)
    gen = torch.Generator(DEV).manual_seed(3)
    k = (k.float() * torch.linspace(0, 2, states, device=DEV)[None, :, None, None]).to(BF16)
    v = ((1 + torch.rand(v.shape, generator=gen, device=DEV) * 0.9) * 2.0**power).to(BF16)
    v[:, :, 1] *= -1
    lengths = [states, states - 1][: len(rows)]
    for x in (q, torch.zeros_like(q)):
        got = attention.cross(torch, x, k, v, starts=counts(rows), lengths=ints(lengths), most=max(rows))
        check(got, x, k, v, counts(rows), ints(lengths))


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside minus infinity"])
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_cross_scores_far_below_zero(attention, rows, beside, dtype):
    """Ten states that all score -2^106, and nothing else seen, or nothing but scores of minus infinity: their values'
    mean. Scores that are equal are off alike, so that only the weights' and the output's roundings count."""
    requests, width, states = len(rows), 64, 4100
    scale = 2.0**96 if dtype is FP16 else 2.0**-10
    q = torch.full((sum(rows), 2, width), 16.0 if dtype is FP16 else 2.0**55, dtype=dtype, device=DEV)
    _, _, v = inputs(1, requests, states, 2, 2, width, dtype, 4)
    for at in (0, 710, 4080):
        k = torch.full((requests, states, 2, width), -math.inf, dtype=dtype, device=DEV)
        k[:, at : at + 10] = -1.0 if dtype is FP16 else -(2.0**55)
        mask = None
        if not beside:
            mask = torch.zeros(requests, states, dtype=torch.bool, device=DEV)
            mask[:, at : at + 10] = True
        got = attention.cross(torch, q, k, v, starts=counts(rows), mask=mask, most=max(rows), scale=scale).double()
        want = v[:, at : at + 10].double().mean(1).repeat_interleave(ints(rows), 0)
        size = v[:, at : at + 10].double().abs().mean(1).repeat_interleave(ints(rows), 0)
        assert ((got - want).abs() <= UNIT[dtype] * want.abs() + (UNIT[dtype] + 2.0**-20) * size).all(), at


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("states", [33, 450, 5000])
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_cross_values_that_are_all_the_type_s_largest(attention, rows, states, dtype):
    """Their mean is the type's largest too: no rounding of weights takes it past that."""
    most = torch.finfo(dtype).max
    q, k, v = inputs(sum(rows), len(rows), states, 4, 2, 64, dtype, states)
    v = torch.full_like(v, most)
    v[..., ::3] *= -1
    got = attention.cross(torch, q, k, v, starts=counts(rows), most=max(rows)).double()
    want = v[0, 0].double().repeat_interleave(2, 0)
    # A weight is off by half a step at the most, and their sum, as a share of it, no more; then the output's half step.
    assert ((got - want).abs() <= (2 * UNIT[dtype] + 2.0**-18) * most).all() and got.isfinite().all()
    # An infinity among them is the mean, and beside one of the other sign NaN.
    v[:, states // 2, 0, 0], v[:, 5, 1, 1], v[:, 6, 1, 1] = math.inf, math.inf, -math.inf
    got = attention.cross(torch, torch.zeros_like(q), k, v, starts=counts(rows), most=max(rows))
    assert (got[:, :2, 0] == math.inf).all() and got[:, 2:, 1].isnan().all() and got[:, :2, 1:].isfinite().all()
