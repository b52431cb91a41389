"""The paged cache of keys and values in 8 bits on gfx950: a step's plan, the write of its tokens, and
attention over what the cache holds.

A page holds `page` tokens of every key head as int8 or E4M3 codes with one float32 scale a page and
head, for keys and for values: value = code · scale. A decode step then reads half the bytes that a
16-bit cache would cost it. Keys stand as `[pages, heads, page, D]`, values transposed as
`[pages, heads, D, page]` (both operands of attention's matrix instructions as they lie).

One step of a model, on one stream:

    plan = kv_cache.plan(torch, table, free, spare, lengths, new, tokens=T, page=cache.page, most=1)
    for each layer:
        q, k = heads.norm_rope(torch, q, k, q_gain, k_gain, cos, sin, plan.positions)
        cache.append(torch, k, v, plan)
        out = cache.attend(torch, q, plan)
    lengths, spare = plan.lengths, plan.spare

Nothing here waits for the GPU, so a step may be captured into a HIP graph (pass `out=plan`, whose
tensors each replay then writes again). A request that ends gives its pages back by writing their
numbers to `free[spare:]` and adding their count to `spare`.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

from cozyq import _dispatch

Tensor = Any
Dtype = Any

OP = "cozy-kv-cache"
#: Tokens a page may hold.
PAGES = (16, 32, 64, 128, 256)
#: Head widths the cache takes.
WIDTHS = (64, 128, 256)


@dataclass(slots=True)
class Plan:
    """A step over a paged cache: `T` rows, the new tokens of `R` requests one request after another.

    `table` int32 `[R, W]`: each request's pages; `starts` `[R + 1]`: its first row; `lengths` `[R]`:
    the tokens it holds after the step; `positions`, `requests`, `slots` `[T]`: a row's position in its
    request, its request and its slot (page · page size + place), 0, -1 and -1 for a row of no request,
    slot -1 where no page was left; `runs` `[N, 4]`: the new tokens of one page each (first row, count,
    page or -1, first place in the page), unused ones last as (0, 0, -1, 0); `spare` `[2]`: free pages
    left, and pages wanted and not got. `most`: the most rows a request has, as far as the host knows
    (0: not at all); attention chooses its kernels by it, and any value is right."""

    page: int
    most: int
    table: Tensor
    starts: Tensor
    lengths: Tensor
    positions: Tensor
    requests: Tensor
    slots: Tensor
    runs: Tensor
    spare: Tensor


def plan(torch: Any, table: Tensor, free: Tensor, spare: Tensor, held: Tensor, new: Tensor, *, tokens: int,
         page: int, most: int = 0, out: Plan | None = None) -> Plan:  # fmt: skip
    """The step in which request r, holding `held[r]` tokens, brings `new[r]` (int32 `[R]` on the GPU):
    `tokens` rows, those past the requests' own belonging to none. Pages that a request does not hold
    yet come off the end of `free` (int32, `spare[0]` of them free) in row order, and their numbers go
    into `table` (int32 `[R, W]`, in place). A request whose rows would pass `tokens` has its count cut
    there. `out`: a plan of the same shape to write again (its `spare` and `lengths` may not be this
    call's inputs). Up to 4000 requests."""
    if most < 0:
        raise ValueError(f"plan: a request has no {most} rows")
    parts = _dispatch.library(_dispatch.card(OP, table)).cache_plan(table, free, spare, held, new, tokens, page, out)
    if out is None:
        return Plan(page, most, table, *parts)
    out.most = most
    return out


def empty(torch: Any, pages: int, heads: int, width: int, *, page: int = 64, dtype: Dtype = None,
          device: Any = "cuda") -> PagedCache:  # fmt: skip
    """A cache of `pages` pages of `page` tokens for `heads` key heads of `width`, in `dtype`
    (torch.int8, the default, or torch.float8_e4m3fn)."""
    dtype = torch.int8 if dtype is None else dtype
    if page not in PAGES or width not in WIDTHS or pages < 1 or heads < 1:
        raise ValueError(f"{OP}: pages of {PAGES} tokens and heads of width {WIDTHS}; got page {page}, width "
                         f"{width}, {pages} pages, {heads} heads")  # fmt: skip
    if dtype is not torch.int8 and dtype is not torch.float8_e4m3fn:
        raise ValueError(f"{OP}: codes are int8 or float8_e4m3fn, not {dtype}")
    codes = torch.zeros(2, pages * heads * page * width, dtype=torch.int8, device=device).view(dtype)
    scales = torch.zeros(2, pages, heads, dtype=torch.float32, device=device)
    return PagedCache(codes[0].view(pages, heads, page, width), codes[1].view(pages, heads, width, page),
                      scales[0], scales[1])  # fmt: skip


@dataclass(slots=True)
class PagedCache:
    """One layer's cache: codes `k` `[pages, heads, page, D]` and `v` `[pages, heads, D, page]` (int8 or
    float8_e4m3fn), float32 scales `k_scale` and `v_scale` `[pages, heads]`. `empty` makes one."""

    k: Tensor
    v: Tensor
    k_scale: Tensor
    v_scale: Tensor

    @property
    def page(self) -> int:
        return int(self.k.shape[2])

    def append(self, torch: Any, k: Tensor, v: Tensor, plan: Plan) -> None:
        """The step's keys and values `[T, heads, D]` (bf16 or fp16; views as `heads.norm_rope` takes
        them) into the pages of `plan.runs`. A page's scale is the largest magnitude among its tokens
        over 127 (int8) or 448 (E4M3), at least 1e-12: a run that begins its page sets it, a later one
        raises it where it must, and what the page holds is then rounded again. An infinity or NaN makes
        its page's scale so, for that head: every query that sees the page is NaN there."""
        index = _dispatch.card(OP, k)
        _dispatch.library(index).cache_append(self, k, v, plan)

    def read(self, torch: Any, pages: Tensor, dtype: Dtype) -> tuple[Tensor, Tensor]:
        """Pages `pages` (int32 `[n]`) as numbers in `dtype` (bf16 or fp16): keys and values, both
        `[n, heads, page, D]`; zeros for a number that is no page of the cache (a plan's -1, say)."""
        index = _dispatch.card(OP, self.k)
        _dispatch.sixteen_bit(OP, torch, dtype)
        return _dispatch.library(index).cache_read(self, pages, dtype)

    def attend(self, torch: Any, q: Tensor, plan: Plan, *, scale: float | None = None, causal: bool = True,
               window: int = 0) -> Tensor:  # fmt: skip
        """Attention of the step's queries `[T, q_heads, D]` (bf16 or fp16; views as
        `heads.norm_rope` takes them) over their requests' pages, `[T, q_heads, D]` in q's type: query
        head h reads key head h // (q_heads / heads). Row t sees its request's tokens up to its own
        position, with a `window` the last `window` of them; without `causal`, all of them. `scale`
        multiplies the scores (None: D^-1/2). A row that sees nothing, or belongs to no request, is 0. A plan
        put together without its rows' slots (an empty tensor) goes by `starts`: q may then have fewer rows than
        that speaks of, or more."""
        index = _dispatch.card(OP, q)
        return _dispatch.library(index).cache_attend(self, q, plan, scale, causal, window)
