"""Attention to an encoder's states (`cozyq.attention.cross`) at the ends of its types, against `oracle/layer.py`; bars
as in test_gpu_cross.py."""

from __future__ import annotations

import pytest
import torch

from test_gpu_cross import BF16, check, counts, inputs
from test_gpu_kv_cache import DEV, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attention():
    from cozyq import attention

    return attention


# One row and a few, two tiles of few rows, part of a tile of many, more than one.
ROWS = [[1, 2], [20], [60, 1], [130, 1], [300]]


@pytest.mark.parametrize("states", [40, 450, 5000])
@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("power", [126, 60, -100])
def test_cross_values_of_any_size(attention, rows, states, power):
    """bf16 values near the type's ends: their weighted means are as large, whatever their sums would be. Scores grow
    along the states, so that the largest is met late."""
    q, k, v = inputs(sum(rows), len(rows), states, 4, 2, 64, BF16, states)
    gen = torch.Generator(DEV).manual_seed(3)
    k = (k.float() * torch.linspace(0, 2, states, device=DEV)[None, :, None, None]).to(BF16)
    v = ((1 + torch.rand(v.shape, generator=gen, device=DEV) * 0.9) * 2.0**power).to(BF16)
    v[:, :, 1] *= -1
    lengths = [states, states - 1][: len(rows)]
    for x in (q, torch.zeros_like(q)):
        got = attention.cross(torch, x, k, v, starts=counts(rows), lengths=ints(lengths), most=max(rows))
        check(got, x, k, v, counts(rows), ints(lengths))
