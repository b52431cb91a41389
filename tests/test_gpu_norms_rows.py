"""GPU test of the residual norm in 8 bits (`cozyq.norms`) over more rows than a launch's one dimension has."""

from __future__ import annotations

import pytest
import torch

from test_gpu_kv_cache import DEV
from test_gpu_norms import E4M3, FP16, check, norms, provider, rows_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes,width,times", [(E4M3, 16, (1 << 20) + 1), (torch.int8, 256, 1 << 15), (torch.int8, 256, (1 << 15) + 1)])
def test_add_rms_of_very_many_rows(norms, codes, width, times):  # noqa: F811
    """2^26 + 64 short rows, of a wave each: 2^32 threads and more; and 2^21 rows and 64 more. Every 64 rows are those 64."""
    x, r, gain = rows_of((64, width), FP16, 41)
    once, total = norms.add_rms(torch, x, r, gain, provider=provider(codes))
    check(once, total, x, r, gain, codes)
    x, r = x.repeat(times, 1), r.repeat(times, 1)
    got, sums = norms.add_rms(torch, x, r, gain, provider=provider(codes), out=r)
    assert sums is r
    assert bool((r.view(times, 64, width) == total).all())
    assert bool((got.payload.view(torch.uint8).view(times, 64, width) == once.payload.view(torch.uint8).view(64, width)).all())
    assert bool((got.scale.view(times, 64) == once.scale.view(64)).all())
