"""Attention over the paged cache at scores far below zero; bars as in test_gpu_kv_cache.py."""

from __future__ import annotations

import pytest
import torch

from test_gpu_kv_cache import DEV, E4M3, UNIT, kv, make_plan  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
@pytest.mark.parametrize("new,length", [(1, 10), (5, 33), (40, 64)])
@pytest.mark.parametrize("width", [64, 256])
def test_attend_scores_far_below_zero(kv, new, length, width, codes):  # noqa: F811
    """Tokens that all score below -2^105: their values' mean. Scores that are equal are off alike, so that only the
    weights' and the output's roundings count."""
    gen = torch.Generator().manual_seed(length)
    k = torch.ones(1, 2, 64, width).to(codes)
    raw = torch.randint(-127, 128, (1, 2, 64, width), generator=gen).float().to(codes)
    v = raw.view(torch.int8).transpose(2, 3).contiguous().view(codes)
    far, one = torch.full((1, 2), 2.0**50), torch.ones(1, 2)
    cache = kv.PagedCache(k.to(DEV), v.to(DEV), far.to(DEV), one.to(DEV))
    plan, _, tokens = make_plan(kv, [[0]], [length], [new], 64, new)
    q = torch.full((tokens, 8, width), -(2.0**52), dtype=torch.bfloat16, device=DEV)
    got = cache.attend(torch, q, plan, causal=False).cpu().double()
    seen = raw[0, :, :length].double().repeat_interleave(4, 0)
    want, size = seen.mean(1), seen.abs().mean(1)
    assert ((got - want).abs() <= UNIT[torch.bfloat16] * want.abs() + (2.0**-11 + 2.0**-12) * size).all()
