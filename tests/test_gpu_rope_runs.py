"""GPU parity of `cozyq.heads.norm_rope` where a wave takes several runs of heads, on one axis and on several, and where
heads are fewer than a wave's places; bars as in test_gpu_kv_cache.py."""

from __future__ import annotations

import pytest
import torch

from oracle import cache as law
from oracle import layer
from test_gpu_kv_cache import DEV, check_rope, rope_inputs

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16

# Two runs in three parts for five; three in two with a last part of two; three with a last run past the heads; one part
# of all runs; 13 heads in two places each; keys that begin within a run; and one head to a wave's places and fewer.
SHAPES = [(1000, 32, 8, 128, 128, BF16), (1400, 32, 8, 128, 128, FP16), (2100, 7, 2, 256, 256, BF16), (5000, 20, 20, 64, 64, FP16),
          (900, 23, 3, 240, 96, BF16), (1700, 13, 5, 96, 96, FP16), (4097, 1, 0, 64, 64, BF16), (9001, 1, 1, 16, 16, FP16),
          (5003, 8, 1, 64, 32, BF16), (70001, 1, 0, 128, 128, FP16), (3, 2, 1, 128, 64, BF16)]  # fmt: skip


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("tokens,heads,k_heads,width,rotated,dtype", SHAPES)
def test_norm_rope_of_many_waves(tokens, heads, k_heads, width, rotated, dtype, interleaved):
    from cozyq import heads as ops

    qkv, cos, sin, positions, gains = rope_inputs(tokens, heads, k_heads, width, rotated, dtype, tokens, rows=997)
    on, gains, c, s = qkv.to(DEV), gains.to(dtype).to(DEV), cos.to(DEV), sin.to(DEV)
    q, k = on[:, :heads], on[:, heads : heads + k_heads] if k_heads else None
    gain = gains[0].contiguous(), gains[1].contiguous() if k_heads else None
    pairs = rotated // 2
    for sections in (None, (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)):
        at, turn = positions, (cos, sin, positions)
        if sections:
            gen = torch.Generator().manual_seed(tokens)
            at = torch.randint(-2, 1000, (3, tokens), generator=gen, dtype=torch.int32)
            turn = (*layer.tables(cos, sin, at, sections, interleaved), None)
        got = ops.norm_rope(torch, q, k, *gain, c, s, at.to(DEV), eps=1e-5, interleaved=interleaved, sections=sections,
                            cycled=interleaved and sections is not None)  # fmt: skip
        assert (got[1] is None) == (k is None)
        for part, x, g in zip(got, (q, k), gains):
            if x is not None:
                check_rope(part, *law.norm_rope(x.cpu(), g.cpu(), *turn, 1e-5, interleaved), dtype)
