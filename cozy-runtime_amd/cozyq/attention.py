"""Attention of a decoder's rows to an encoder's states of another length on gfx950 (`cozyq_cross_attend`): to an image's
or a recording's from the text about it, to a text's from the image or video that it describes.

The states' keys and values are dense in bf16 or fp16, `[requests, states, heads, D]`: one projection of the encoder's
output, padded to the longest. Attention to a decoder's own tokens is `kv_cache.PagedCache.attend`.
"""

from __future__ import annotations

from typing import Any

from cozyq import _dispatch

Tensor = Any

OP = "cozy-attention"


def cross(torch: Any, q: Tensor, k: Tensor, v: Tensor, *, starts: Tensor | None = None, lengths: Tensor | None = None,
          mask: Tensor | None = None, most: int = 0, scale: float | None = None) -> Tensor:  # fmt: skip
    """Rows `q` `[T, q_heads, D]` over the states `k`, `v` `[R, S, heads, D]` of their requests, `[T, q_heads, D]` in q's
    type (bf16 or fp16): softmax(`scale` · q·k) · v (None: D^-1/2), query head h reading key head h // (q_heads / heads).
    Request r's rows are `starts[r]` to `starts[r + 1]` (int32 `[R + 1]`, ascending, a plan's; None: T / R each). A row
    sees the first `lengths[r]` states of its request (int32 `[R]`; None: all S) that `mask` has (bool `[R, S]`, True:
    seen; None: all); where that is none, or of a row of no request, the result is 0. What is not seen reaches no
    result, whatever it holds. `starts`, `lengths` and `mask` are read on the GPU, so that a step may be captured into a
    HIP graph and replayed over others. `most`: the most rows a request has, as far as the host knows (0: not at all);
    kernels are chosen by it, and any value is right, but 0 beside `starts` takes all rows for one request's: single
    tokens of 24 requests over up to 1600 states then take 37 us instead of 29. Scores, the softmax and sums are float32
    (scores past its range are infinities); each state's weight is rounded to q's type before it multiplies v. D is a multiple of 8 up to 256. q, k and v may be views (of one
    projection's buffer, say) whose last axis is dense and whose other strides and address are multiples of 16 bytes.
    A workspace comes from torch's allocator where states are split over workgroups. Results carry no gradient."""
    index = _dispatch.card(OP, q)
    return _dispatch.library(index).cross_attend(q, k, v, starts, lengths, mask, most, scale)
