"""GPU tests of the paged cache where rows, plans and requests do not fit one another: steps of more rows than
the requests bring, queries of another number of rows than the plan's, requests that hold more than their row of
the table names.

Bars as in test_gpu_kv_cache.py: the output's one rounding, and of Σ p·|v| the weights' 2^-11 and the exponents'
2^-12."""

from __future__ import annotations

import math
import random

import pytest
import torch

from test_gpu_kv_cache import DEV, E4M3, UNIT, check_plan, filled, ints, kv, make_plan  # noqa: F401

pytestmark = pytest.mark.gpu


def expected(q, value, table, starts, lengths, page, causal=True, window=0):
    """float64 on the GPU, a request at a time: (out, Σ p·|v|). A request's rows are its last tokens."""
    tokens, q_heads, width = q.shape
    heads = value.shape[2]
    group = q_heads // heads
    out = torch.zeros(tokens, q_heads, width, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    for r, length in enumerate(lengths):
        first, last = starts[r], min(starts[r + 1], tokens)
        if last <= first or length <= 0:
            continue
        numbers = torch.tensor(table[r][: -(-length // page)])
        k, v = (x[numbers].to(DEV).double().transpose(0, 1).reshape(heads, -1, width)[:, :length] for x in value)
        position = length - (starts[r + 1] - first) + torch.arange(last - first, device=DEV)
        at = torch.arange(length, device=DEV)
        hidden = torch.zeros(last - first, length, dtype=torch.bool, device=DEV)
        if causal:
            hidden |= at > position[:, None]
        if window:
            hidden |= at <= position[:, None] - window
        for h in range(heads):
            mine = slice(h * group, (h + 1) * group)
            x = q[first:last, mine].to(DEV).double().reshape(-1, width)
            score = (x @ k[h].T.contiguous() * width**-0.5).view(last - first, group, length)
            p = score.masked_fill(hidden[:, None], -math.inf).softmax(-1).nan_to_num(0.0).view(-1, length)
            out[first:last, mine] = (p @ v[h]).view(last - first, group, width)
            size[first:last, mine] = (p @ v[h].abs()).view(last - first, group, width)
    return out, size


def over_nan(cache, q, plan, **how):
    """attend's result, in memory that held NaN before the call."""
    torch.cuda.empty_cache()
    junk = [torch.full(q.shape, math.nan, dtype=q.dtype, device=DEV) for _ in range(4)]
    where = {x.data_ptr() for x in junk}
    del junk
    out = cache.attend(torch, q, plan, **how)
    assert out.data_ptr() in where
    return out


def check(kv, lengths, new, page, q_heads, heads, width, codes, dtype, tokens, lead=0, most=None, columns=0, window=0,
          causal=True):  # fmt: skip
    """Every row against the formula; rows of no request, `lead` of them before the first request's, are 0."""
    seed = sum(lengths) + 31 * sum(new) + page + width
    cache, table, value = filled(kv, lengths, page, heads, width, codes, seed)
    table = [row + [-1] * (columns - len(row)) for row in table]
    plan, starts, _ = make_plan(kv, table, lengths, new, page, max(new) if most is None else most)
    starts = [lead + s for s in starts]
    plan.starts = ints(starts)
    q = torch.randn(tokens, q_heads, width, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    got = over_nan(cache, q, plan, window=window, causal=causal)
    assert (got[:lead] == 0).all() and (got[starts[-1] :] == 0).all()
    want, size = expected(q, value, table, starts, lengths, page, causal, window)
    bar = UNIT[dtype] * want.abs() + (2.0**-11 + 2.0**-12) * size + (2.0**-25 if dtype is torch.float16 else 0)
    assert ((got.double() - want).abs() <= bar).all()


# ------------------------------------------------------------------- rows of no request

#: Decode steps of a fixed number of rows of which some requests are gone, and prompts shorter than their step.
PADDED = {
    "40 of 64, long": dict(lengths=[200 + 17 * i for i in range(40)], new=[1] * 40, tokens=64, columns=40, most=1),
    "1 of 8, long": dict(lengths=[30000], new=[1], tokens=8, most=1),
    "1 of 64, long": dict(lengths=[30000], new=[1], tokens=64, most=1),
    "32 of 64": dict(lengths=[4000] * 32, new=[1] * 32, tokens=64, columns=100, most=1),
    "8 of 64, a short table": dict(lengths=[200], new=[8], tokens=64, columns=4, most=0),
    "574 of 704, many rows": dict(lengths=[3774], new=[574], tokens=704),
    "300 of 2000, many rows": dict(lengths=[3000, 70, 900], new=[100, 1, 199], tokens=2000),
    "none of 700": dict(lengths=[500, 90], new=[0, 0], tokens=700, most=0),
}


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
@pytest.mark.parametrize("lead", [0, 37])
@pytest.mark.parametrize("step", list(PADDED), ids=list(PADDED))
def test_rows_of_no_request_are_zero(kv, step, lead, codes):  # noqa: F811
    how = dict(PADDED[step])
    how["tokens"] += lead
    check(kv, page=64, q_heads=32, heads=8, width=64, codes=codes, dtype=torch.bfloat16, lead=lead, **how)


@pytest.mark.parametrize("seed", range(24))
def test_rows_of_no_request_are_zero_in_drawn_steps(kv, seed):  # noqa: F811
    rng = random.Random(seed)
    q_heads, heads, width = rng.choice(((32, 8, 128), (16, 16, 64), (28, 4, 128), (64, 8, 128), (16, 2, 256), (8, 1, 64)))
    requests = rng.choice((1, 2, 7, 30, 70))
    held = [rng.randrange(1, 40000 // requests) for _ in range(requests)]
    new = [rng.choice((0, 1, 1, 1, 4)) for _ in held] if rng.random() < 0.6 else [rng.randrange(400 // requests + 2) for _ in held]
    page, lead = rng.choice((16, 64, 256)), rng.choice((0, 0, 1, 90))
    check(kv, [h + n for h, n in zip(held, new)], new, page, q_heads, heads, width, rng.choice((torch.int8, E4M3)),
          rng.choice((torch.bfloat16, torch.float16)), lead + sum(new) + rng.choice((1, 9, 60, 700)), lead,
          rng.choice((None, 0)), columns=rng.choice((0, 600)), window=rng.choice((0, 0, 300)))  # fmt: skip


# ------------------------------------------------------- queries of other rows than the plan's


@pytest.mark.parametrize("new,tokens", [([5, 1, 9], 10), ([5, 1, 9], 3), ([40, 300], 200), ([40, 300], 17)],
                         ids=["few", "few, first", "many", "many, first"])  # fmt: skip
@pytest.mark.parametrize("window", [0, 50])
def test_rows_past_the_queries_move_no_position(kv, new, tokens, window):  # noqa: F811
    """A step cut short: the rows that are there see what they see in the whole step."""
    lengths = [n + 60 * (i + 1) for i, n in enumerate(new)]
    cache, table, value = filled(kv, lengths, 16, 4, 64, torch.int8, 5)
    plan, starts, whole = make_plan(kv, table, lengths, new, 16, max(new))
    q = torch.randn(whole, 32, 64, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    got = cache.attend(torch, q[:tokens], plan, window=window)
    want, size = expected(q[:tokens], value, table, starts, lengths, 16, window=window)
    assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-12) * size).all()


def test_queries_of_another_number_of_rows_are_refused(kv):  # noqa: F811
    cache = kv.empty(torch, 4, 2, 64, page=16, device=DEV)
    plan = kv.plan(torch, ints([[-1, -1]]), ints([0, 1]), ints([2]), ints([0]), ints([20]), tokens=20, page=16)
    q = torch.zeros(21, 4, 64, dtype=torch.bfloat16, device=DEV)
    for rows in (0, 1, 19, 21):
        with pytest.raises(ValueError, match="20 rows"):
            cache.attend(torch, q[:rows], plan)
    assert cache.attend(torch, q[:20], plan).shape == (20, 4, 64)


# ------------------------------------------------------------------------ a plan's last pages


@pytest.mark.parametrize("held,new", [([40], [1]), ([40, 5], [0, 0]), ([32, 5, 70], [1, 12, 30]), ([47, 31, 0], [2, 2, 60]),
                                      ([2**30 - 256] * 40, [1, 0, 16, 17] * 10)])  # fmt: skip
@pytest.mark.parametrize("spare", [0, 1, 9])
def test_pages_wanted_are_those_of_new_tokens(kv, held, new, spare):  # noqa: F811
    """Requests that hold more than their row of the table names want a page where a new token begins one."""
    table = [[2 * i, 2 * i + 1] if n >= 32 else [2 * i, -1] if n else [-1, -1] for i, n in enumerate(held)]
    check_plan(kv, table, list(range(100, 109)), spare, held, new, sum(new) + 2, 16)


def test_plan_of_the_most_rows(kv):  # noqa: F811
    """2^30 rows, the first two requests asking for more than there are: their counts add up past 31 bits."""
    rows = 2**30
    got = kv.plan(torch, ints([[-1, -1], [7, -1], [-1, -1]]), ints([3, 4]), ints([2]), ints([0, 9, 0]),
                  ints([rows, 2**31 - 1, 5]), tokens=rows, page=16)  # fmt: skip
    assert got.starts.tolist() == [0, rows, rows, rows] and got.lengths.tolist() == [rows, 9, 0]
    assert got.runs[:3].tolist() == [[0, 16, 4, 0], [16, 16, 3, 0], [32, 16, -1, 0]] and got.table.tolist()[0] == [4, 3]
    assert got.slots[:33].tolist() == [*range(64, 80), *range(48, 64), -1]
    assert got.positions[-1].item() == rows - 1 and got.requests[-1].item() == 0
    assert got.spare.tolist() == [0, rows // 16 - 2]


# ------------------------------------------------------------------------------- arguments


@pytest.mark.parametrize("window", [2**31 - 1, 2**31, 2**32, 2**32 + 5, 2**40])
@pytest.mark.parametrize("new", [[1, 2], [150, 90]], ids=["few", "many"])
def test_windows_past_32_bits_hide_nothing(kv, new, window):  # noqa: F811
    lengths = [200, 700]
    cache, table, _ = filled(kv, lengths, 16, 2, 64, torch.int8, 7)
    plan, _, tokens = make_plan(kv, table, lengths, new, 16, max(new))
    q = torch.randn(tokens, 16, 64, generator=torch.Generator().manual_seed(8)).bfloat16().to(DEV)
    assert torch.equal(cache.attend(torch, q, plan, window=window), cache.attend(torch, q, plan, window=2**20))


@pytest.mark.parametrize("new", [[5, 2], [150, 90]], ids=["few", "many"])
def test_windows_of_any_size_over_lengths_below_the_rows(kv, new):  # noqa: F811
    """Rows at positions below zero see nothing, and those at zero and above what they would without a window."""
    lengths = [1, 2]
    cache, table, _ = filled(kv, lengths, 16, 2, 64, torch.int8, 9)
    plan, _, tokens = make_plan(kv, table, lengths, new, 16, max(new))
    q = torch.randn(tokens, 16, 64, generator=torch.Generator().manual_seed(10)).bfloat16().to(DEV)
    plain = cache.attend(torch, q, plan)
    assert (plain[: new[0] - 1] == 0).all() and (plain[new[0] - 1] != 0).any() and (plain[-1] != 0).any()
    for window in (2**31 - 1, 2**31 - 2, 2**30):
        assert torch.equal(cache.attend(torch, q, plan, window=window), plain)


def test_caches_of_no_pages_or_heads_are_refused(kv):  # noqa: F811
    for pages, heads in ((0, 2), (2, 0)):
        codes = torch.zeros(pages, heads, 64, 64, dtype=torch.int8, device=DEV)
        scale = torch.zeros(pages, heads, device=DEV)
        cache = kv.PagedCache(codes, codes, scale, scale)
        plan = kv.plan(torch, ints([[-1]]), ints([0]), ints([0]), ints([0]), ints([2]), tokens=2, page=64)
        x = torch.zeros(2, max(heads, 1), 64, dtype=torch.bfloat16, device=DEV)
        for call in (lambda: cache.append(torch, x[:, :heads], x[:, :heads], plan), lambda: cache.attend(torch, x, plan),
                     lambda: cache.read(torch, ints([0]), torch.bfloat16)):  # fmt: skip
            with pytest.raises(ValueError, match="cache"):
                call()


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
@pytest.mark.parametrize("apart", [0, 64, 109])
@pytest.mark.parametrize("new", [[1, 3], [150, 90]], ids=["few", "many"])
def test_value_scales_far_apart_share_one_denominator(kv, new, apart, codes):  # noqa: F811
    """Pages whose value scales are 2^`apart` apart in turn, equal keys: the small ones' tokens weigh as much."""
    lengths, page = [400, 1700], 16
    cache, table, value = filled(kv, lengths, page, 4, 64, codes, 15)
    cache.k_scale.zero_()
    value[0].nan_to_num_(0.0).zero_()
    for row in table:
        for i, number in enumerate(n for n in row if n >= 0):
            power = 2.0 ** (apart - 40 if i % 3 == 1 else -40)
            cache.v_scale[number] *= power
            value[1, number] *= power
    plan, starts, tokens = make_plan(kv, table, lengths, new, page, max(new))
    q = torch.randn(tokens, 32, 64, generator=torch.Generator().manual_seed(16)).bfloat16().to(DEV)
    got = cache.attend(torch, q, plan)
    want, size = expected(q, value, table, starts, lengths, page)
    assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-12) * size).all()
