"""Queries and keys between the QKV projection and attention, on gfx950: each head's RMS norm and its
rotation to the token's position in one pass (`cozyq_head_norm_rope`).

The reference's counterpart (`kernels/csrc/norm/rms_rope.cu`) lies outside its quantized-linear path.
"""

from __future__ import annotations

from typing import Any

from cozyq import _dispatch

Tensor = Any

OP = "cozy-heads"


def norm_rope(torch: Any, q: Tensor, k: Tensor | None, q_gain: Tensor | None, k_gain: Tensor | None,
              cos: Tensor | None, sin: Tensor | None, positions: Tensor | None = None, *,
              eps: float | None = 1e-6, interleaved: bool = False) -> tuple[Tensor, Tensor | None]:  # fmt: skip
    """Every head of `q` `[T, heads, D]` and `k` `[T, k_heads, D]` (None: queries alone), bf16 or fp16,
    in float32 and rounded once: times rsqrt(mean(x²) + `eps`) and its gain `[D]` (float32 or x's type;
    None: 1; `eps` None: no norm), then its first 2·`cos.shape[1]` elements rotated in pairs, halves
    (i, i + R/2) or, `interleaved`, neighbours (2i, 2i + 1): (a, b) -> (a·cos − b·sin, b·cos + a·sin).
    `cos` and `sin` are float32 `[rows, R/2]` (None: no rotation), read at `positions[t]` (int32 `[T]`;
    None: row t; a position outside the table reads its nearest row). D and R are multiples of 16, D up
    to 256. q and k may be views (of one QKV buffer, say) whose last axis is dense and whose other
    strides and address are multiples of 16 bytes; the results are new and contiguous."""
    return _dispatch.library(_dispatch.card(OP, q)).head_norm_rope(q, k, q_gain, k_gain, cos, sin, positions, eps, interleaved)
