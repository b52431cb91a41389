"""The residual stream between a quantized model's linears on gfx950: a linear's output added to the stream, the RMS
norm of the sum, and that in 8 bits as the next linear's operand, in one pass (`cozyq_add_rms`).

    x = int8_linear.gemm(torch, operand, *layer.out, None, torch.bfloat16)
    operand, stream = norms.add_rms(torch, x, stream, layer.gain, provider=operands.INT8_CONVROT)
    y = int8_linear.gemm(torch, operand, *layer.up, None, torch.bfloat16)

The reference's producer prologue (`internal/int8_linear.py:308-357`, here `operands.int8_rows`) norms and quantizes
rows that are summed already.
"""

from __future__ import annotations

from typing import Any

from cozyq import _dispatch
from cozyq.operands import INT8_CONVROT, ROWWISE_FP8, PreQuantized

Tensor = Any

OP = "cozy-norms"
#: Which operands a norm writes, and whether they are E4M3.
PROVIDERS = {INT8_CONVROT: False, ROWWISE_FP8: True}


def add_rms(torch: Any, x: Tensor, residual: Tensor | None, gain: Tensor | None, *, provider: str = INT8_CONVROT,
            eps: float = 1e-6, out: Tensor | None = None) -> tuple[PreQuantized, Tensor]:  # fmt: skip
    """`(operand, total)`: total = `x` + `residual` (`[..., K]`, bf16 or fp16, one shape and type) rounded to their
    type, and the rows total · rsqrt(mean(total²) + `eps`) · `gain` (`[K]`, float32 or x's type; None: 1) in 8 bits, in
    float32 throughout: `INT8_CONVROT` rotated int8 (K % 256 == 0), `ROWWISE_FP8` E4M3 (K % 16 == 0), K up to 32768, as
    the operand that `int8_linear.gemm`, `fp8_linear.gemm` and the leaves read. Without a `residual` total is x itself.
    `out`: where total goes, a dense tensor like x; it may be `x` or `residual`, whole. A row that holds a NaN or an
    infinity has the scale NaN. Results carry no gradient."""
    index = _dispatch.activation_card(OP, torch, x)
    fp8 = PROVIDERS.get(provider)
    if fp8 is None:
        raise ValueError(f"{OP}: operands are {', '.join(PROVIDERS)}, not {provider!r}")
    codes, scale, total = _dispatch.library(index).add_rms(x, residual, gain, fp8, eps, out)
    return PreQuantized(codes, scale, tuple(x.shape), provider), total
