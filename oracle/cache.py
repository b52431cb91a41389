"""The laws of the attention side, restated for the CPU: the plan of a step over a paged cache in
Python integers, the cache's codes and scales in float32 as the kernels round them, and the head norm,
the rotation and attention in float64."""

from __future__ import annotations

import math

import torch

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FLOOR = 1e-12


def plan(table, free, spare, held, new, tokens: int, page: int) -> dict:
    """One request after another, one token after another."""
    table = [list(map(int, row)) for row in table]
    requests, width = len(table), len(table[0])
    free, left, short = [int(f) for f in free], min(int(spare), len(free)), 0
    starts, lengths, positions, owners, slots, runs = [0], [], [], [], [], []
    for r in range(requests):
        length, count = max(0, int(held[r])), max(0, int(new[r]))
        count = min(count, tokens - starts[-1])
        for i in range(count):
            index, place = divmod(length + i, page)
            if place == 0:  # a page that the request does not hold yet
                number = -1
                if index < width:
                    if left > 0:
                        left -= 1
                        number = free[left]
                    table[r][index] = number
                short += number < 0
            number = table[r][index] if index < width else -1
            if i == 0 or place == 0:
                runs.append([starts[-1] + i, 0, number, place])
            runs[-1][1] += 1
            positions.append(length + i)
            owners.append(r)
            slots.append(number * page + place if number >= 0 else -1)
        starts.append(starts[-1] + count)
        lengths.append(length + count)
    rest = tokens - len(positions)
    most = min(tokens, tokens // page + 2 * requests)
    return {"table": table, "starts": starts, "lengths": lengths, "positions": positions + [0] * rest,
            "requests": owners + [-1] * rest, "slots": slots + [-1] * rest,
            "runs": runs + [[0, 0, -1, 0]] * (most - len(runs)), "spare": [left, short]}  # fmt: skip


def _codes(x: torch.Tensor, dtype) -> torch.Tensor:
    """float32 -> codes by their values; 0 for NaN."""
    most = MOST[dtype]
    x = torch.where(x.isnan(), 0.0, x).clamp(-most, most)
    return x.round() if dtype is torch.int8 else x.to(dtype).float()


def append(codes: torch.Tensor, scale: torch.Tensor, new: torch.Tensor, runs, dtype) -> None:
    """Writes the runs' tokens of `new` `[T, heads, D]` into the pages' values `codes` (float32 code
    values, `[pages, heads, page, D]`) and `scale` `[pages, heads]`, in place, each step in float32."""
    most = torch.tensor(MOST[dtype])
    for row, count, number, place in runs:
        if count <= 0 or not 0 <= number < codes.shape[0]:
            continue
        x = new[row : row + count].float().transpose(0, 1)
        before = scale[number].clone() if place else torch.zeros(scale.shape[1])
        reach = torch.maximum(x.abs().amax((1, 2)) / most, torch.tensor(FLOOR))
        after = torch.maximum(before, reach)
        grown = after.view(torch.int32) != before.view(torch.int32)
        if place:
            ratio = torch.where(grown, before / after, 1.0)[:, None, None]
            codes[number] = torch.where(grown[:, None, None], _codes(codes[number] * ratio, dtype), codes[number])
        else:
            codes[number] = 0.0
        codes[number, :, place : place + count] = _codes(x / after[:, None, None], dtype)
        scale[number] = after


def norm_rope(x, gain, cos, sin, positions, eps, interleaved: bool):
    """float64: (result, the magnitude its rounding errors scale with)."""
    x = x.double()
    if eps is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        if gain is not None:
            x = x * gain.double()
    size = x.abs()
    if cos is not None:
        rows = (torch.arange(x.shape[0]) if positions is None else positions.long()).clamp(0, cos.shape[0] - 1)
        c, s = cos.double()[rows][:, None], sin.double()[rows][:, None]
        half = cos.shape[1]
        out = x.clone()
        size = x.abs().clone()
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
        x = out
    return x, size


def attend(q, k, v, table, starts, lengths, page: int, scale=None, causal=True, window=0):
    """float64 over values k, v `[pages, heads, page, D]`: (out `[T, q_heads, D]`, Σ p·|v| beside it)."""
    tokens, q_heads, width = q.shape
    pages, heads = k.shape[:2]
    scale = width**-0.5 if scale is None else scale
    out = torch.zeros(tokens, q_heads, width, dtype=torch.float64)
    size = torch.zeros_like(out)
    for r in range(len(lengths)):
        first, last, length = int(starts[r]), int(starts[r + 1]), int(lengths[r])
        if last <= first or length <= 0:
            continue
        held = [int(n) for n in table[r][: -(-length // page)]]
        held += [-1] * (-(-length // page) - len(held))
        there = torch.tensor([0 <= n < pages for n in held]).repeat_interleave(page)[:length]
        number = torch.tensor([n if 0 <= n < pages else 0 for n in held])
        kk = k[number].double().transpose(0, 1).reshape(heads, -1, width)[:, :length]
        vv = v[number].double().transpose(0, 1).reshape(heads, -1, width)[:, :length]
        at = torch.arange(length)
        for t in range(first, last):
            position = length - (last - first) + t - first
            seen = there.clone()
            if causal:
                seen &= at <= position
            if window:
                seen &= at > position - window
            if not seen.any():
                continue
            score = q[t].double().view(heads, -1, width) @ kk[:, seen].transpose(1, 2) * scale
            p = (score - score.amax(-1, keepdim=True)).exp()
            p = torch.where(score.isnan().any(-1, keepdim=True), math.nan, p / p.sum(-1, keepdim=True))
            out[t] = (p @ vv[:, seen]).view(q_heads, width)
            size[t] = (p @ vv[:, seen].abs()).view(q_heads, width)
    return out, size
