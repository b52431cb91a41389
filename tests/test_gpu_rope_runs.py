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

# Waves enough for several runs each: two of three, the last short; three of one part; two of two on one axis and four of
# one on several; three of three; the same with a last run past the heads; keys that begin within a run. Then heads fewer
# than a wave's places, whose waves hold several tokens' (nine and one of 16 places, two of 64, one of eight).
SHAPES = [(3300, 32, 8, 128, 128, BF16), (6001, 20, 20, 64, 64, FP16), (4200, 28, 4, 128, 64, BF16), (1900, 64, 8, 128, 128, FP16),
          (2400, 23, 3, 240, 96, BF16), (5600, 13, 5, 96, 96, FP16), (5601, 7, 2, 256, 256, BF16), (1000, 32, 8, 128, 128, FP16),
          (5003, 8, 1, 64, 32, BF16), (4097, 1, 0, 64, 64, BF16), (9001, 1, 1, 16, 16, FP16), (70001, 1, 0, 128, 128, FP16),
          (3, 2, 1, 128, 64, BF16)]  # fmt: skip


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("tokens,heads,k_heads,width,rotated,dtype", SHAPES)
def test_norm_rope_of_many_waves(tokens, heads, k_heads, width, rotated, dtype, interleaved):
    from cozyq import heads as ops

    qkv, cos, sin, positions, gains = rope_inputs(tokens, heads, k_heads, width, rotated, dtype, tokens, rows=997)
    on, gains, cos, sin, positions = qkv.to(DEV), gains.to(dtype).to(DEV), cos.to(DEV), sin.to(DEV), positions.to(DEV)
    q, k = on[:, :heads], on[:, heads : heads + k_heads] if k_heads else None
    gain = gains[0].contiguous(), gains[1].contiguous() if k_heads else None
    pairs = rotated // 2
    for sections in (None, (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)):
        at, turn = positions, (cos, sin, positions)
        if sections:
            gen = torch.Generator().manual_seed(tokens)
            at = torch.randint(-2, 1000, (3, tokens), generator=gen, dtype=torch.int32).to(DEV)
            turn = (*layer.tables(cos, sin, at, sections, interleaved), None)
        got = ops.norm_rope(torch, q, k, *gain, cos, sin, at, eps=1e-5, interleaved=interleaved, sections=sections,
                            cycled=interleaved and sections is not None)  # fmt: skip
        assert (got[1] is None) == (k is None)
        for part, x, g in zip(got, (q, k), gains):
            if x is not None:
                want, size = law.norm_rope(x, g, *turn, 1e-5, interleaved)
                check_rope(part, want.cpu(), size.cpu(), dtype)


def test_norm_rope_of_one_short_head_of_very_many_tokens():
    """As many tokens as a launch has waves, and more: 2^32 threads would be one too many, a lane a head is not."""
    from cozyq import heads as ops

    qkv, cos, sin, _, _ = rope_inputs(64, 1, 0, 16, 16, BF16, 31)
    q, cos, sin = qkv.to(DEV), cos.to(DEV), sin.to(DEV)
    at, times = torch.arange(64, dtype=torch.int32, device=DEV) * 2, (1 << 20) + 1
    once = ops.norm_rope(torch, q, None, None, None, cos, sin, at)[0]
    check_rope(once, *law.norm_rope(qkv, None, cos.cpu(), sin.cpu(), at.cpu(), 1e-6, False), BF16)
    got = ops.norm_rope(torch, q.repeat(times, 1, 1), None, None, None, cos, sin, at.repeat(times))[0]
    assert bool((got.view(times, 64, 1, 16) == once).all())
