"""The residual norm in 8 bits, positions on several axes and attention to an encoder's states, from their formulas in
64 bits (no reference counterpart: parity is with the mathematics). Test infrastructure, on any device."""

from __future__ import annotations

import math

import torch

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FLOOR = 1e-12


def hadamard256() -> torch.Tensor:
    """The regular Hadamard H4⊗H4⊗H4⊗H4 over 16, of norm 1, float64."""
    h = torch.ones(4, 4, dtype=torch.float64) - 2 * torch.eye(4, dtype=torch.float64).flip(0)
    for _ in range(3):
        h = torch.kron(h, torch.ones(4, 4, dtype=torch.float64) - 2 * torch.eye(4, dtype=torch.float64).flip(0))
    return h / 16


def add_rms(x, residual, gain, codes, eps: float):
    """(total in x's type, the rows before their rounding to codes over their scale, the scale [rows, 1], and beside the
    rows the mean magnitude of what each was summed from): float64."""
    total = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    n = total.double()
    n = n / (n.square().mean(-1, keepdim=True) + eps).sqrt()
    if gain is not None:
        n = n * gain.double()
    summed = n.abs()
    if codes is torch.int8:
        h = hadamard256().to(x.device)
        shape = n.shape
        n = (n.view(-1, 256) @ h).view(shape)
        summed = (summed.view(-1, 256) @ h.abs()).view(shape)
    scale = (n.abs().amax(-1, keepdim=True) / MOST[codes]).clamp(min=FLOOR)
    return total, n, scale, summed


def axis_of_pairs(sections, cycled: bool) -> list[int]:
    """The axis of each pair: runs of `sections`, or in turns, axis a > 0 having a, a + axes, .. and axis 0 the rest."""
    if not cycled:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axis = [0] * sum(sections)
    for a, n in enumerate(sections):
        for i in range(n if a else 0):
            axis[a + len(sections) * i] = a
    return axis


def tables(cos, sin, positions, sections, cycled: bool):
    """Each token's own cosines and sines [tokens, pairs] of positions [axes, tokens], the nearest row for one outside
    the tables."""
    axis = axis_of_pairs(sections, cycled)
    row = positions.long().clamp(0, cos.shape[0] - 1)[axis].T
    return cos.gather(0, row), sin.gather(0, row)


def cross(q, k, v, starts, lengths, mask=None, scale=None):
    """float64: (out [tokens, heads, D], Σ p·|v| beside it). Rows of no request, and rows that see nothing, are 0."""
    tokens, heads, width = q.shape
    requests, states, kv_heads = k.shape[:3]
    scale = width**-0.5 if scale is None else scale
    out = torch.zeros(tokens, heads, width, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for b in range(requests):
        first, last = max(0, int(starts[b])), min(int(starts[b + 1]), tokens)
        length = min(max(int(lengths[b]), 0), states)
        seen = torch.arange(length, device=q.device)
        if mask is not None:
            seen = seen[mask[b, :length]]
        if last <= first or not len(seen):
            continue
        kk, vv = (x[b, seen].double().transpose(0, 1).contiguous() for x in (k, v))
        group = heads // kv_heads
        for h in range(heads):
            score = q[first:last, h].double() @ kk[h // group].T.contiguous() * scale
            p = (score - score.amax(-1, keepdim=True)).exp()
            p = torch.where(score.isnan().any(-1, keepdim=True), math.nan, p / p.sum(-1, keepdim=True))
            out[first:last, h] = p @ vv[h // group]
            size[first:last, h] = p @ vv[h // group].abs()
    return out, size
