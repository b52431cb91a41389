"""GPU parity of the paged 8-bit cache (`cozyq.kv_cache`) and of the head norm and rotation
(`cozyq.heads`) against `oracle/cache.py`.

Bars, by what each operator rounds:
- plans are equal; codes and scales are bit-exact to the float32 law;
- norm_rope: one rounding to the 16-bit type of float32 arithmetic: u·|y| + 16·2^-24·(|a| + |b|), with
  u = 2^-8 (bf16) or 2^-11 (fp16), and a subnormal half step;
- attend: u·|y| for the one rounding, and of Σ p·|v| the weights' f16 rounding, 2^-11 at the most, with
  2^-12 for the exponents' (a score of magnitude 64·log2(e) in float32 is off by 2^-18 at the most, the
  sums and the power of two by less)."""

from __future__ import annotations

import math
import random

import pytest
import torch

from oracle import cache as law

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def kv():
    from cozyq import kv_cache

    return kv_cache


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------ plan


def check_plan(kv, table, free, spare, held, new, tokens, page, out=None):
    t = ints(table)
    got = kv.plan(torch, t, ints(free), ints([spare]), ints(held), ints(new), tokens=tokens, page=page, out=out)
    want = law.plan(table, free, spare, held, new, tokens, page)
    for name, value in want.items():
        assert getattr(got, name).tolist() == value, name
    assert got.table is t
    return got


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("requests,tokens", [(1, 1), (1, 0), (3, 700), (65, 65), (257, 1000), (1100, 5003), (4000, 4100)])
def test_plan(kv, requests, tokens, page):
    rng = random.Random(requests * 1000 + page)
    held = [rng.choice((0, 1, page - 1, page, page + 1, rng.randrange(5 * page))) for _ in range(requests)]
    new = [0] * requests
    for _ in range(max(0, tokens - rng.choice((0, 0, 3)))):
        new[rng.randrange(requests)] += 1
    if requests > 2:  # one takes most, some bring none
        new[1] += new[0] + new[2]
        new[0] = new[2] = 0
    width = max(-(-(h + n) // page) for h, n in zip(held, new)) + 1
    numbers = list(range(7, 7 + sum(-(-(h + n) // page) for h, n in zip(held, new)) + 4))
    rng.shuffle(numbers)
    table = [[numbers.pop() if i < -(-h // page) else -1 for i in range(width)] for h in held]
    check_plan(kv, table, numbers, len(numbers), held, new, tokens, page)


def test_plan_without_enough_pages_columns_or_rows(kv):
    table = [[3, -1], [-1, -1], [8, 9]]
    check_plan(kv, table, [1, 2], 2, [16, 0, 30], [40, 20, 5], 65, 16)  # free pages and columns run out
    check_plan(kv, table, [1, 2], 0, [16, 0, 30], [1, 1, 1], 3, 16)  # none free
    check_plan(kv, table, [1, 2], -4, [16, 0, 30], [1, 1, 1], 3, 16)
    check_plan(kv, table, [1, 2], 9, [16, 0, 30], [1, 1, 1], 3, 16)  # more spare than the list is long
    check_plan(kv, table, [4, 5, 6, 7], 4, [16, -5, 30], [2, -3, 9], 7, 16)  # negatives; the rows end early
    check_plan(kv, table, [4, 5, 6, 7], 4, [16, 0, 30], [2**31 - 1, 2**31 - 1, 1], 9, 16)  # sums past 32 bits


@pytest.mark.parametrize("page", [16, 256])
def test_plan_of_counts_past_any_cache(kv, page):
    # What a request may hold is cut at 2^30 - 256: its sums stay below 2^31, its rows get no page, others' do.
    t = ints([[3, 4], [5, -1]])
    got = kv.plan(torch, t, ints([8, 9]), ints([2]), ints([2**31 - 1, page]), ints([3, 2]), tokens=5, page=page)
    held = 2**30 - 256
    assert got.lengths.tolist() == [held + 3, page + 2]
    assert got.positions.tolist() == [held, held + 1, held + 2, page, page + 1]
    assert got.slots.tolist() == [-1, -1, -1, 9 * page, 9 * page + 1]
    assert got.runs.tolist()[:2] == [[0, 3, -1, 0], [3, 2, 9, 0]]
    assert t.tolist() == [[3, 4], [5, 9]] and int(got.spare[0]) == 1


def test_plan_written_again_and_in_a_graph(kv):
    """`out` takes the next step's plan; captured, each replay gives the eager plan's answer."""
    table, free = [[5, -1, -1], [-1, -1, -1]], [0, 1, 2, 3, 4]
    first = check_plan(kv, table, free, 5, [10, 0], [6, 16], 22, 16)
    t, f, spare, held, new = first.table, ints(free), first.spare.clone(), first.lengths.clone(), ints([1, 1])
    second = kv.plan(torch, t, f, spare, held, new, tokens=2, page=16)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kv.plan(torch, t, f, spare, held, new, tokens=2, page=16, out=second)
    for step in ([1, 1], [0, 2], [2, 0]):
        new.copy_(ints(step))
        now = law.plan(t.tolist(), free, int(spare[0]), held.tolist(), step, 2, 16)
        graph.replay()
        torch.cuda.synchronize()
        for name, value in now.items():
            assert getattr(second, name).tolist() == value, (step, name)
        held.copy_(second.lengths)
        spare.copy_(second.spare)
    with pytest.raises(ValueError, match="inputs"):
        kv.plan(torch, t, f, second.spare, held, new, tokens=2, page=16, out=second)
    with pytest.raises(ValueError, match="out"):
        kv.plan(torch, t, f, spare, held, new, tokens=3, page=16, out=second)


def test_plan_refusals(kv):
    t, one = ints([[0, 1]]), ints([1])
    for bad in (dict(table=t.long()), dict(table=t[0]), dict(held=ints([1, 2])), dict(new=one.float()), dict(page=24),
                dict(tokens=-1), dict(free=t), dict(most=-1), dict(table=ints([[0]] * 4001), held=ints([0] * 4001), new=ints([0] * 4001))):  # fmt: skip
        a = dict(table=t, free=one, spare=one, held=one, new=one, tokens=1, page=16, most=0) | bad
        with pytest.raises(ValueError):
            kv.plan(torch, a["table"], a["free"], a["spare"], a["held"], a["new"], tokens=a["tokens"], page=a["page"], most=a["most"])


# --------------------------------------------------------------------------- norm and rotation


def rope_inputs(tokens, heads, k_heads, width, rotated, dtype, seed, rows=None):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, heads + 2 * k_heads, width, generator=gen) * torch.exp2(
        torch.randint(-6, 7, (tokens, heads + 2 * k_heads, 1), generator=gen)
    )
    qkv = qkv.to(dtype)
    rows = rows or 2 * tokens + 3
    angle = torch.rand(rows, rotated // 2, generator=gen) * 6.28
    positions = torch.randint(0, rows, (tokens,), generator=gen, dtype=torch.int32)
    gains = 1 + 0.2 * torch.randn(2, width, generator=gen)
    return qkv, angle.cos(), angle.sin(), positions, gains


def check_rope(got, want, size, dtype):
    error = (got.cpu().double() - want).abs()
    bar = UNIT[dtype] * want.abs() + 16 * 2.0**-24 * size + (2.0**-25 if dtype is torch.float16 else 0)
    assert got.is_contiguous() and (error <= bar).all(), float((error / bar.clamp(min=1e-30)).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("tokens,heads,k_heads,width,rotated", [
    (1, 1, 1, 16, 16), (1, 32, 8, 128, 128), (7, 5, 3, 64, 32), (33, 12, 12, 80, 80), (130, 3, 1, 96, 48),
    (19, 7, 2, 256, 256), (601, 6, 2, 128, 64), (5, 4, 4, 192, 160), (3, 2, 2, 240, 16)])  # fmt: skip
def test_norm_rope(tokens, heads, k_heads, width, rotated, interleaved, dtype):
    from cozyq import heads as ops

    qkv, cos, sin, positions, gains = rope_inputs(tokens, heads, k_heads, width, rotated, dtype, tokens + width)
    on = qkv.to(DEV)
    q, k = on[:, :heads], on[:, heads : heads + k_heads]
    for wide in (False, True):
        g = gains if wide else gains.to(dtype)
        got = ops.norm_rope(torch, q, k, g[0].contiguous().to(DEV), g[1].contiguous().to(DEV), cos.to(DEV), sin.to(DEV),
                            positions.to(DEV), eps=1e-5, interleaved=interleaved)  # fmt: skip
        for part, x, gain in zip(got, (q, k), g):
            check_rope(part, *law.norm_rope(x.cpu(), gain, cos, sin, positions, 1e-5, interleaved), dtype)


def test_norm_rope_parts_left_out():
    """No norm, no gain, no table, no positions, no keys, none of the rows; positions off the table."""
    from cozyq import heads as ops

    dtype = torch.bfloat16
    qkv, cos, sin, positions, gains = rope_inputs(9, 3, 2, 64, 64, dtype, 5)
    on, c, s = qkv.to(DEV), cos.to(DEV), sin.to(DEV)
    q, k = on[:, :3], on[:, 3:5]
    got = ops.norm_rope(torch, q, k, None, None, None, None, eps=None)
    assert torch.equal(got[0], q) and torch.equal(got[1], k)
    got, none = ops.norm_rope(torch, q, None, gains[0].contiguous().to(DEV), None, None, None)
    assert none is None
    check_rope(got, *law.norm_rope(q.cpu(), gains[0], None, None, None, 1e-6, False), dtype)
    got = ops.norm_rope(torch, q, k, None, None, c, s, eps=None)[1]
    check_rope(got, *law.norm_rope(k.cpu(), None, cos, sin, None, None, False), dtype)
    far = positions.clone()
    far[0], far[1] = -5, 10**6
    got = ops.norm_rope(torch, q, k, None, None, c, s, far.to(DEV))[0]
    check_rope(got, *law.norm_rope(q.cpu(), None, cos, sin, far, 1e-6, False), dtype)
    got = ops.norm_rope(torch, q[:0], k[:0], None, None, c, s)
    assert got[0].shape == (0, 3, 64) and got[1].shape == (0, 2, 64)
    wild = q.clone()
    wild[0, 0, 3], wild[1, 1, 2], wild[2] = math.inf, math.nan, 0
    got = ops.norm_rope(torch, wild, None, None, None, c, s)[0].cpu()
    want = law.norm_rope(wild.cpu(), None, cos, sin, None, 1e-6, False)[0]
    assert got[0, 0].isnan().any() and got[1, 1].isnan().all() and (got[2] == 0).all()
    keep = torch.ones(9, 3, dtype=torch.bool)
    keep[0, 0] = keep[1, 1] = False
    check_rope(got[keep], want[keep], want[keep].abs() + 10, dtype)


def test_norm_rope_refusals():
    from cozyq import heads as ops

    qkv, cos, sin, positions, gains = (x.to(DEV) for x in rope_inputs(4, 2, 2, 64, 64, torch.bfloat16, 6))
    q, k, g = qkv[:, :2], qkv[:, 2:4], gains[0].contiguous()
    good = dict(q=q, k=k, qg=None, kg=None, cos=cos, sin=sin, positions=positions, eps=1e-6)
    for bad in (dict(q=q.float()), dict(k=k.half()), dict(k=k[:3]), dict(q=q[..., :40]), dict(q=q[..., 1:]), dict(q=q[0]),
                dict(qg=g.half()), dict(qg=g[:32]), dict(qg=g, kg=g.bfloat16()), dict(qg=g, eps=None), dict(sin=None),
                dict(cos=cos.half()), dict(cos=cos[:, :20], sin=sin[:, :20]), dict(positions=positions.long()),
                dict(positions=positions[:2]), dict(positions=None, cos=cos[:3].contiguous(), sin=sin[:3].contiguous()),
                dict(cos=torch.cat((cos, cos), 1), sin=torch.cat((sin, sin), 1)), dict(cos=cos.cpu()),
                dict(q=q.transpose(0, 2))):  # fmt: skip
        a = good | bad
        with pytest.raises(ValueError):
            ops.norm_rope(torch, a["q"], a["k"], a["qg"], a["kg"], a["cos"], a["sin"], a["positions"], eps=a["eps"])


# ------------------------------------------------------------------------------ append and read


def values_of(cache):
    """Code values as float32 [pages, heads, page, D] on the CPU, keys and values."""
    k, v = cache.k.cpu(), cache.v.cpu()
    return k.float(), v.float().transpose(2, 3).contiguous()


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.int32), b.contiguous().view(torch.int32))


def loud(shape, gen, dtype):
    x = torch.randn(shape, generator=gen)
    return (x * torch.exp2(torch.randint(-3, 4, shape[:2], generator=gen))[..., None]).to(dtype)


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("page,width,heads", [(16, 64, 1), (32, 128, 3), (64, 128, 2), (128, 64, 2), (256, 256, 1)])
def test_append_steps_bit_exact(kv, page, width, heads, dtype, codes):
    """Several steps over one cache: pages begun, filled, gone past, and begun by a later request."""
    gen = torch.Generator().manual_seed(page + width)
    cache = kv.empty(torch, 40, heads, width, page=page, dtype=codes, device=DEV)
    want = [torch.zeros(40, heads, page, width), torch.zeros(40, heads, page, width)]
    scales = [torch.zeros(40, heads), torch.zeros(40, heads)]
    requests = 4
    table = torch.full((requests, 9), -1, dtype=torch.int32, device=DEV)
    free, spare, held = ints(list(range(40))), ints([40]), ints([0] * requests)
    for new in ([1, page, 3, 0], [1, 1, 2 * page - 3, 2], [page - 2, 0, 1, 1], [1, 1, 1, page + 5], [7, 1, 0, 1]):
        tokens = sum(new) + 2  # the last rows belong to none
        plan = kv.plan(torch, table, free, spare, held, ints(new), tokens=tokens, page=page)
        kv_new = loud((tokens, 2 * heads, width), gen, dtype)
        on = kv_new.to(DEV)
        cache.append(torch, on[:, :heads], on[:, heads:], plan)
        runs = plan.runs.tolist()
        for i, got in enumerate(values_of(cache)):
            law.append(want[i], scales[i], kv_new[:, i * heads : (i + 1) * heads], runs, codes)
            assert torch.equal(got, want[i])
        assert same_bits(cache.k_scale.cpu(), scales[0]) and same_bits(cache.v_scale.cpu(), scales[1])
        held, spare = plan.lengths, plan.spare
    numbers = plan.runs[:, 2].contiguous()
    back = cache.read(torch, numbers, dtype)
    for got, value, scale in zip(back, want, scales):
        expect = (value * scale[..., None, None]).to(dtype)[numbers.cpu().long().clamp(min=0)]
        expect[numbers.cpu() < 0] = 0
        assert torch.equal(got.cpu(), expect)


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
def test_append_of_zeros_tiny_huge_and_not_finite_tokens(kv, codes):
    """The scale's floor, magnitudes at the ends of bf16, and infinities and NaN, which stay with their
    page, head and tensor while every code stays finite."""
    page, width, heads = 16, 64, 4
    cache = kv.empty(torch, 4, heads, width, page=page, dtype=codes, device=DEV)
    x = torch.randn(20, 2 * heads, width, generator=torch.Generator().manual_seed(9)).bfloat16()
    x[:, 0] = 0
    x[:, 1] *= 2.0**-120
    x[:, 2] *= 2.0**120
    x[2, 3, 5], x[18, 4, 7], x[1, 5, 0] = math.inf, math.nan, -math.inf
    plan = kv.plan(torch, ints([[-1, -1]]), ints([0, 1, 2]), ints([3]), ints([0]), ints([20]), tokens=20, page=page)
    on = x.to(DEV)
    cache.append(torch, on[:, :heads], on[:, heads:], plan)
    for i, (got, scale) in enumerate(zip(values_of(cache), (cache.k_scale.cpu(), cache.v_scale.cpu()))):
        want, scales = torch.zeros(4, heads, page, width), torch.zeros(4, heads)
        law.append(want, scales, x[:, i * heads : (i + 1) * heads], plan.runs.tolist(), codes)
        assert got.isfinite().all() and torch.equal(scale.isfinite(), scales.isfinite()) and torch.equal(scale.isnan(), scales.isnan())
        fine = scales.isfinite()
        assert torch.equal(got[fine], want[fine]) and same_bits(scale[fine], scales[fine])
    assert cache.k_scale[2, 0] == 1e-12 or cache.k_scale[1, 0] == 1e-12


def test_append_skips_runs_without_a_page(kv):
    cache = kv.empty(torch, 2, 1, 64, page=16, device=DEV)
    x = torch.ones(40, 1, 64, dtype=torch.bfloat16, device=DEV)
    plan = kv.plan(torch, ints([[-1, -1, -1]]), ints([99, 1]), ints([2]), ints([0]), ints([40]), tokens=40, page=16)
    assert plan.runs[:3, 2].tolist() == [1, 99, -1] and plan.spare.tolist() == [0, 1]
    cache.append(torch, x, x, plan)
    assert (cache.k[1] == 127).all() and (cache.k[0] == 0).all() and (cache.k_scale[0] == 0).all()
    k, v = cache.read(torch, ints([1, 99, -1]), torch.float16)
    assert (k[0] == 1).all() and (v[0] == 1).all() and (k[1:] == 0).all() and (v[1:] == 0).all()


def test_append_and_read_refusals(kv):
    cache = kv.empty(torch, 2, 2, 64, page=16, device=DEV)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    plan = kv.plan(torch, ints([[0]]), ints([1]), ints([1]), ints([0]), ints([4]), tokens=4, page=16)
    other = kv.plan(torch, ints([[0]]), ints([1]), ints([1]), ints([0]), ints([4]), tokens=4, page=32)
    for k, v, p in ((x.float(), x, plan), (x, x.half(), plan), (x[:3], x[:3], plan), (x[:, :1], x, plan), (x, x[..., :32], plan),
                    (x, x, other), (x.transpose(1, 2), x, plan), (x.cpu(), x, plan)):  # fmt: skip
        with pytest.raises(ValueError):
            cache.append(torch, k, v, p)
    with pytest.raises(ValueError):
        cache.read(torch, ints([0]).long(), torch.bfloat16)
    with pytest.raises(ValueError):
        cache.read(torch, ints([0]), torch.float32)
    bad = kv.PagedCache(cache.k, cache.k, cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError):
        bad.read(torch, ints([0]), torch.bfloat16)
    bad = kv.PagedCache(cache.k, cache.v, cache.k_scale[:1], cache.v_scale)
    with pytest.raises(ValueError):
        bad.append(torch, x, x, plan)


# ------------------------------------------------------------------------------------ attend


def filled(kv, lengths, page, heads, width, codes, seed, spread=0, extra=3):
    """A cache of random codes and scales (`spread`: powers of two between pages' scales) and a table of
    shuffled pages; bytes past a request's tokens hold anything, NaN codes among them."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + extra
    order = torch.randperm(pages, generator=gen).tolist()
    columns = max(1, max(counts) + 1)
    table = [[order.pop() if i < c else -1 for i in range(columns)] for c in counts]
    shape = (2, pages, heads, page, width)
    if codes is torch.int8:
        raw = torch.randint(-127, 128, shape, generator=gen).to(torch.int8)
    else:
        raw = (torch.randn(shape, generator=gen) * 60).clamp(-448, 448).to(E4M3)
    scale = (0.5 + torch.rand(2, pages, heads, generator=gen)) / (64 if codes is torch.int8 else 60)
    scale = scale * torch.exp2(torch.randint(-spread, spread + 1, (2, pages, heads), generator=gen))
    value = raw.float() * scale[..., None, None]
    junk = raw.view(torch.int8)
    for r, n in enumerate(lengths):
        if n % page:
            number, place = table[r][n // page], n % page
            junk[:, number, :, place:] = torch.randint(-128, 128, (2, heads, page - place, width), generator=gen).to(torch.int8)
            if codes is E4M3:
                junk[:, number, :, place] = 127  # NaN
            value[:, number, :, place:] = math.nan
    k = raw[0].contiguous().to(DEV)
    v = raw[1].view(torch.int8).transpose(2, 3).contiguous().view(codes).to(DEV)
    cache = kv.PagedCache(k, v, scale[0].contiguous().to(DEV), scale[1].contiguous().to(DEV))
    return cache, table, value


def make_plan(kv, table, lengths, new, page, most, tokens=None):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    tokens = starts[-1] if tokens is None else tokens
    nothing = torch.zeros(0, dtype=torch.int32, device=DEV)
    plan = kv.Plan(page=page, most=most, table=ints(table), starts=ints(starts), lengths=ints(lengths), positions=nothing,
                   requests=nothing, slots=nothing, runs=nothing, spare=nothing)  # fmt: skip
    return plan, starts, tokens


def check_attend(kv, lengths, new, page, q_heads, heads, width, codes, dtype, window=0, causal=True, most=None, spread=0,
                 tokens=None, scale=None):  # fmt: skip
    seed = sum(lengths) + 31 * sum(new) + page + width
    cache, table, value = filled(kv, lengths, page, heads, width, codes, seed, spread)
    plan, starts, tokens = make_plan(kv, table, lengths, new, page, max(new) if most is None else most, tokens)
    q = torch.randn(tokens, q_heads + 1, width, generator=torch.Generator().manual_seed(seed)).to(dtype)[:, 1:]
    got = cache.attend(torch, q.to(DEV), plan, window=window, causal=causal, scale=scale).cpu()
    want, size = law.attend(q, value[0], value[1], table, starts, lengths, page, scale, causal, window)
    assert got.dtype == dtype and got.shape == (tokens, q_heads, width)
    error = (got.double() - want).abs()
    bar = UNIT[dtype] * want.abs() + (2.0**-11 + 2.0**-12) * size + (2.0**-25 if dtype is torch.float16 else 0)
    assert got.isfinite().all() and (error <= bar).all(), float((error / bar.clamp(min=1e-30)).max())
    return got


BOTH = pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])


@BOTH
@pytest.mark.parametrize("q_heads,heads,width", [(4, 4, 64), (8, 2, 128), (7, 1, 64), (6, 2, 256), (32, 2, 128), (64, 1, 64)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attend_one_token_a_request(kv, page, q_heads, heads, width, codes):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 130, 257, 700]
    check_attend(kv, lengths, [1] * len(lengths), page, q_heads, heads, width, codes, torch.bfloat16)


@BOTH
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("q_heads,heads,width", [(4, 4, 64), (8, 2, 128), (3, 1, 256), (28, 4, 64)])
@pytest.mark.parametrize("new", [[2, 5, 1, 8], [3, 0, 70, 33], [40, 129, 1, 0], [1, 200, 17, 65]], ids=lambda n: "-".join(map(str, n)))
def test_attend_several_tokens_a_request(kv, new, q_heads, heads, width, dtype, codes):
    held = [0, 100, 31, 64]
    check_attend(kv, [h + n for h, n in zip(held, new)], new, 32, q_heads, heads, width, codes, dtype)


@pytest.mark.parametrize("window", [1, 15, 64, 100, 5000])
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 3, 50], [150, 0, 200]], ids=lambda n: "-".join(map(str, n)))
def test_attend_window(kv, new, window):
    held = [300, 5, 64]
    check_attend(kv, [h + n for h, n in zip(held, new)], new, 64, 8, 2, 64, torch.int8, torch.float16, window=window)


@pytest.mark.parametrize("new", [[1, 3], [70, 130]], ids=["few", "many"])
def test_attend_all_tokens(kv, new):
    """Without causal: every row sees all of its request, a request of no tokens nothing."""
    check_attend(kv, [90, 200], new, 16, 6, 3, 64, E4M3, torch.bfloat16, causal=False)
    got = check_attend(kv, [0, 200], new, 16, 6, 3, 64, E4M3, torch.bfloat16, causal=False)
    assert (got[: new[0]] == 0).all()


@pytest.mark.parametrize("most", [0, 1, 4, 64, 4096])
def test_attend_results_hold_for_any_hint(kv, most):
    check_attend(kv, [300, 40, 513, 7], [1, 40, 130, 2], 32, 8, 2, 64, torch.int8, torch.bfloat16, most=most, tokens=180)


@BOTH
@pytest.mark.parametrize("new", [[1, 1], [66, 140]], ids=["few", "many"])
def test_attend_pages_of_very_different_scales(kv, new, codes):
    """Pages 2^24 apart in scale: what dominates a row and what its denominator counts differ."""
    check_attend(kv, [700, 1300], new, 16, 4, 2, 64, codes, torch.float16, spread=12, scale=2.0**-14)


#: Steps of so many rows over so many heads that the kernel for many rows takes them: a whole tile and parts of
#: one, a request of one token beside, contexts past the steps that one workgroup takes, none at all.
MANY = [([1500, 40, 3], [150, 1, 33]), ([0, 2100, 17], [260, 1, 0]), ([1200], [201])]


@BOTH
@pytest.mark.parametrize("page,dtype", [(16, torch.float16), (64, torch.bfloat16), (256, torch.bfloat16)], ids=["16", "64", "256"])
@pytest.mark.parametrize("q_heads,heads,width", [(32, 4, 64), (32, 4, 128), (32, 4, 256), (33, 3, 128)])
@pytest.mark.parametrize("held,new", MANY, ids=["beside", "begins", "alone"])
def test_attend_many_rows(kv, held, new, q_heads, heads, width, page, dtype, codes):
    check_attend(kv, [h + n for h, n in zip(held, new)], new, page, q_heads, heads, width, codes, dtype, tokens=sum(new) + 3)


@pytest.mark.parametrize("window", [1, 17, 64, 300, 5000])
@pytest.mark.parametrize("width", [64, 128])
def test_attend_many_rows_with_a_window(kv, width, window):
    held, new = [1500, 40, 3], [150, 1, 33]
    check_attend(kv, [h + n for h, n in zip(held, new)], new, 32, 32, 4, width, torch.int8, torch.bfloat16, window=window)


@BOTH
def test_attend_many_rows_of_all_tokens_and_of_very_different_scales(kv, codes):
    lengths, new = [400, 0, 1300], [140, 2, 5]
    got = check_attend(kv, lengths, new, 32, 48, 6, 64, codes, torch.bfloat16, causal=False)
    assert (got[140:142] == 0).all()
    check_attend(kv, [700, 1300], [66, 140], 16, 32, 4, 128, codes, torch.float16, spread=12, scale=2.0**-14)


@BOTH
@pytest.mark.parametrize("width", [64, 128, 256])
def test_attend_many_rows_over_missing_and_not_finite_pages(kv, width, codes):
    lengths, new, page = [1250, 90], [160, 1], 16
    cache, table, value = filled(kv, lengths, page, 5, width, codes, 13)
    for index in (3, 5, 11, 74):
        table[0][index] = (-1, 10**6, -7, -1)[index % 4]
    for index, bad in ((70, math.nan), (71, math.inf)):  # tokens 1120 .. 1151
        cache.v_scale[table[0][index]] = bad
        cache.k_scale[table[0][index + 2]] = bad  # 1152 .. 1183
    plan, starts, tokens = make_plan(kv, table, lengths, new, page, 160)
    q = torch.randn(tokens, 40, width, generator=torch.Generator().manual_seed(14)).bfloat16()
    got = cache.attend(torch, q.to(DEV), plan).cpu()
    want, size = law.attend(q, value[0], value[1], table, starts, lengths, page)
    sees = torch.zeros(tokens, 40, dtype=torch.bool)
    sees[30:160] = True  # request 0's rows from position 1120 on
    assert torch.equal(got.isnan().all(-1), sees) and torch.equal(got.isnan().any(-1), sees)
    error = (got.double() - want).abs()
    assert (error[~sees] <= (2.0**-8 * want.abs() + 2.0**-10 * size)[~sees]).all()
    got = cache.attend(torch, q.to(DEV), plan, window=20).cpu()  # the last rows are past the pages and their window
    for t in range(160):
        position = 1090 + t
        sees[t] = position >= 1120 and position - 20 < 1183
    assert torch.equal(got.isnan().all(-1), sees)


def test_attend_many_rows_is_the_same_every_time_and_in_a_graph(kv):
    lengths, new = [3000, 5, 900], [200, 1, 1]
    cache, table, _ = filled(kv, lengths, 64, 4, 128, torch.int8, 31)
    plan, _, tokens = make_plan(kv, table, lengths, new, 64, 200)
    q = torch.randn(tokens, 32, 128, generator=torch.Generator().manual_seed(32)).bfloat16().to(DEV)
    first = cache.attend(torch, q, plan)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = cache.attend(torch, q, plan)
    for _ in range(4):
        assert torch.equal(cache.attend(torch, q, plan), first)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, first)


def test_attend_rows_of_no_request_and_missing_pages(kv):
    for new in ([1, 2], [90, 5]):
        got = check_attend(kv, [100, 200], new, 16, 4, 2, 64, torch.int8, torch.bfloat16, tokens=sum(new) + 5)
        assert (got[sum(new) :] == 0).all()
        # Entries that are no page: not seen; a request whose every entry is none sees nothing.
        cache, table, value = filled(kv, [100, 200], 16, 2, 64, torch.int8, 3)
        table[0] = [-1] * len(table[0])
        table[1][3], table[1][5], table[1][11] = -1, 10**6, -7
        plan, starts, tokens = make_plan(kv, table, [100, 200], new, 16, max(new))
        q = torch.randn(tokens, 4, 64, generator=torch.Generator().manual_seed(4)).bfloat16()
        got = cache.attend(torch, q.to(DEV), plan).cpu()
        want, size = law.attend(q, value[0], value[1], table, starts, [100, 200], 16)
        assert (got[: new[0]] == 0).all()
        assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-10 * size).all()
        # More tokens than the table's rows have pages for: those past it are not seen.
        short = kv.Plan(page=16, most=max(new), table=ints([row[:4] for row in table]), starts=plan.starts, lengths=plan.lengths,
                        positions=plan.positions, requests=plan.requests, slots=plan.slots, runs=plan.runs, spare=plan.spare)  # fmt: skip
        got = cache.attend(torch, q.to(DEV), short).cpu()
        want, size = law.attend(q, value[0], value[1], [row[:4] for row in table], starts, [100, 200], 16)
        assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-10 * size).all()


@pytest.mark.parametrize("new", [[1, 2], [90, 5], [300, 150]], ids=["one", "few", "many"])
def test_attend_lengths_past_any_table(kv, new):
    # Steps end where the table's row does, so that such a call is as short as one over full rows.
    cache, table, value = filled(kv, [96, 192], 16, 2, 64, torch.int8, 61)
    plan, starts, tokens = make_plan(kv, table, [2**31 - 1] * 2, new, 16, max(new))
    q = torch.randn(tokens, 8, 64, generator=torch.Generator().manual_seed(62)).bfloat16()
    got = cache.attend(torch, q.to(DEV), plan, causal=False).cpu()
    want, size = law.attend(q, value[0], value[1], table, starts, [96, 192], 16, None, False)
    error = (got.double() - want).abs()
    assert (error <= UNIT[torch.bfloat16] * want.abs() + (2.0**-11 + 2.0**-12) * size).all()
    assert (cache.attend(torch, q.to(DEV), plan, window=40) == 0).all()


@BOTH
@pytest.mark.parametrize("kind", ["keys", "values"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new", [[1, 1], [150, 40]], ids=["few", "many"])
def test_attend_not_finite_pages_reach_only_the_rows_that_see_them(kv, new, bad, kind, codes):
    page = 16
    lengths = [200, 90]
    cache, table, value = filled(kv, lengths, page, 2, 64, codes, 11)
    scale = cache.k_scale if kind == "keys" else cache.v_scale
    for index in (7, 8, 9):  # tokens 112 .. 159 of request 0, key head 1
        scale[table[0][index], 1] = bad
        value[0 if kind == "keys" else 1, table[0][index], 1] = math.nan
    plan, starts, tokens = make_plan(kv, table, lengths, new, page, max(new))
    q = torch.randn(tokens, 4, 64, generator=torch.Generator().manual_seed(12)).bfloat16()
    got = cache.attend(torch, q.to(DEV), plan).cpu()
    sees = torch.zeros(tokens, 4, dtype=torch.bool)
    for t in range(new[0]):
        sees[t, 2:] = 200 - new[0] + t >= 112
    assert torch.equal(got.isnan().any(-1), sees) and torch.equal(got.isnan().all(-1), sees)
    want, size = law.attend(q, value[0], value[1], table, starts, lengths, page)
    error = (got.double() - want).abs()
    assert (error[~sees] <= (2.0**-8 * want.abs() + 2.0**-10 * size)[~sees]).all()
    got = cache.attend(torch, q.to(DEV), plan, window=30).cpu()  # rows past the pages and their window
    for t in range(new[0]):
        position = 200 - new[0] + t
        sees[t, 2:] = position >= 112 and position - 30 < 159
    assert torch.equal(got.isnan().all(-1), sees)


def test_attend_query_magnitudes(kv):
    """Rows of zeros, at the ends of bf16's range, and not finite ones, which stay NaN alone."""
    lengths = [70, 40]
    cache, table, value = filled(kv, lengths, 16, 1, 64, torch.int8, 21)
    plan, starts, tokens = make_plan(kv, table, lengths, [8, 1], 16, 8)
    q = torch.randn(tokens, 2, 64, generator=torch.Generator().manual_seed(22)).bfloat16()
    q[0], q[1], q[2], q[3, 0, 5], q[4, 1, 6] = 0, q[1] * 2.0**-120, q[2] * 2.0**40, math.nan, math.inf
    got = cache.attend(torch, q.to(DEV), plan).cpu()
    want, size = law.attend(q, value[0], value[1], table, starts, lengths, 16)
    wild = torch.zeros(tokens, 2, dtype=torch.bool)
    wild[3, 0] = wild[4, 1] = True
    assert torch.equal(got.isnan().all(-1), wild) and torch.equal(got.isnan().any(-1), wild)
    # A score of 2^40·64 leaves one token; its float32 rounding cannot change which, the gap is larger.
    assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-10 * size)[~wild].all()


@BOTH
def test_attend_past_32_bit_offsets(kv, codes):
    """A cache of more than 2^31 bytes a tensor, the request's pages at its end."""
    page, heads, width = 128, 8, 128
    pages = 2**31 // (page * heads * width) + 40
    cache = kv.empty(torch, pages, heads, width, page=page, dtype=codes, device=DEV)
    gen = torch.Generator().manual_seed(5)
    table = ints([list(range(pages - 1, pages - 9, -1))])
    x = torch.randn(900, 2 * heads, width, generator=gen).bfloat16().to(DEV)
    plan = kv.plan(torch, ints([[-1] * 8]), table[0].flip(0).contiguous(), ints([8]), ints([0]), ints([900]), tokens=900, page=page)
    cache.append(torch, x[:, :heads], x[:, heads:], plan)
    k, v = cache.read(torch, plan.table[0].contiguous(), torch.bfloat16)
    assert (k.float() - 0).abs().sum() > 0
    q = torch.randn(2, 16, width, generator=gen).bfloat16()
    last, starts, _ = make_plan(kv, plan.table.tolist(), [900], [2], page, 2)
    got = cache.attend(torch, q.to(DEV), last).cpu()
    mine = plan.table[0].tolist()
    values = [(values.float() * s[..., None, None]).cpu() for values, s in (
        (cache.k[mine], cache.k_scale[mine]), (cache.v[mine].view(torch.int8).transpose(2, 3).contiguous().view(codes), cache.v_scale[mine]))]  # fmt: skip
    want, size = law.attend(q, values[0], values[1], [list(range(8))], starts, [900], page)
    assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-10 * size).all()
    near = (k.cpu().double() - values[0].double()).abs() <= 2.0**-8 * values[0].abs()
    assert near.all()


def test_attend_is_the_same_every_time_and_on_another_stream(kv):
    lengths, new = [3000, 5, 900], [1, 1, 1]
    cache, table, _ = filled(kv, lengths, 64, 2, 128, torch.int8, 31)
    plan, _, tokens = make_plan(kv, table, lengths, new, 64, 1)
    q = torch.randn(tokens, 8, 128, generator=torch.Generator().manual_seed(32)).bfloat16().to(DEV)
    first = cache.attend(torch, q, plan)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        assert torch.equal(cache.attend(torch, q, plan), first)
    with torch.cuda.stream(stream):
        other = cache.attend(torch, q, plan)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, first)


@pytest.mark.parametrize("new", [[1, 1, 1], [30, 1, 200]], ids=["few", "many"])
def test_attend_in_a_graph(kv, new):
    """A captured step, replayed over changing lengths with eager work between, equals the eager call."""
    lengths = [700, 64, 400]
    cache, table, _ = filled(kv, lengths, 32, 2, 64, torch.int8, 41)
    plan, _, tokens = make_plan(kv, table, lengths, new, 32, max(new))
    q = torch.randn(tokens, 8, 64, generator=torch.Generator().manual_seed(42)).bfloat16().to(DEV)
    cache.attend(torch, q, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cache.attend(torch, q, plan)
    for shorter in (0, 13, 0, 40):
        plan.lengths.copy_(ints([n - shorter if n > 300 else n for n in lengths]))
        q.add_(0.25)
        want = cache.attend(torch, q, plan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_attend_refusals(kv):
    cache, table, _ = filled(kv, [40], 16, 2, 64, torch.int8, 51)
    plan, _, _ = make_plan(kv, table, [40], [2], 16, 2)
    other, _, _ = make_plan(kv, table, [40], [2], 32, 2)
    wide, _, _ = make_plan(kv, table, [40], [1, 1], 16, 2)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q.transpose(0, 1).transpose(1, 2)),
                dict(plan=other), dict(plan=wide), dict(window=-1), dict(window=4, causal=False),
                dict(q=torch.zeros(2, 2 * 65, 64, dtype=torch.bfloat16, device=DEV)), dict(q=q.cpu())):  # fmt: skip
        a = dict(q=q, plan=plan, window=0, causal=True) | bad
        with pytest.raises(ValueError):
            cache.attend(torch, a["q"], a["plan"], window=a["window"], causal=a["causal"])
    assert cache.attend(torch, q[:0], make_plan(kv, table, [40], [0], 16, 0)[0]).shape == (0, 4, 64)


# -------------------------------------------------------------------------------- a whole layer


@BOTH
def test_a_layer_decodes_as_it_prefills(kv, codes):
    """Quantized projections around the operators: a prompt in one step and the same prompt in chunks and
    single tokens give outputs that agree within the cache's own error (a page's scale may grow later in
    the chunked run, one more half step of its codes)."""
    from cozyq import heads as ops
    from cozyq import int8_linear
    from oracle import laws

    hidden, q_heads, heads, width, page, length = 512, 8, 2, 64, 32, 75
    gen = torch.Generator().manual_seed(61)
    data, scale = laws.int8_weight_rotated(torch.randn((q_heads + 2 * heads) * width, hidden, generator=gen) * 0.05, 256)
    data, scale = data.to(DEV), scale.to(DEV)
    x = torch.randn(length, hidden, generator=gen).bfloat16().to(DEV)
    angle = torch.arange(128)[:, None] * 10000.0 ** (-torch.arange(width // 2) / (width // 2))
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    outs = []
    for split in ([75], [40, 30, 1, 1, 1, 1, 1]):
        cache = kv.empty(torch, 6, heads, width, page=page, dtype=codes, device=DEV)
        table, held, spare = ints([[-1] * 4]), ints([0]), ints([6])
        free, parts, at = ints(list(range(6))), [], 0
        for n in split:
            plan = kv.plan(torch, table, free, spare, held, ints([n]), tokens=n, page=page, most=n)
            qkv = int8_linear.linear(torch, x[at : at + n], data, scale, None, torch.bfloat16).view(n, -1, width)
            q, k = ops.norm_rope(torch, qkv[:, :q_heads], qkv[:, q_heads : q_heads + heads], None, None, cos, sin, plan.positions)
            cache.append(torch, k, qkv[:, q_heads + heads :], plan)
            parts.append(cache.attend(torch, q, plan))
            held, spare, at = plan.lengths, plan.spare, at + n
        outs.append(torch.cat(parts).float())
    # Keys and values hold 7 (int8, of the page's largest) or 4 bits: a few hundredths of the output.
    rel = (outs[0] - outs[1]).norm() / outs[0].norm()
    assert rel < (0.02 if codes is torch.int8 else 0.08), float(rel)


def test_the_decoding_example_replays_what_it_does_eagerly():
    """`examples/decode.py`: prompts, then tokens from a recorded step, against the same steps run eagerly in
    a second server: the same kernels on the same numbers, so the same bits, over page boundaries."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "decode.py"
    spec = importlib.util.spec_from_file_location("decode_example", path)
    example = importlib.util.module_from_spec(spec)
    import sys

    sys.modules["decode_example"] = example
    spec.loader.exec_module(example)
    shape = dict(layers=2, requests=3, q_heads=8, kv_heads=2, width=64, page=16, pages=24, longest=96)
    lengths, steps = [30, 16, 1], 20
    gen = torch.Generator("cuda").manual_seed(71)
    prompt = torch.randn(sum(lengths), 512, generator=gen, device=DEV).bfloat16()
    tokens = torch.randn(steps, 3, 512, generator=gen, device=DEV).bfloat16()
    a, b = example.Server(**shape), example.Server(**shape)
    assert torch.equal(a.prompt(prompt, lengths), b.prompt(prompt, lengths))
    x, y, graph = a.recorded_step()
    one = torch.ones(3, dtype=torch.int32, device=DEV)
    # The recorded server has run its step once before it was recorded: the second one does so too.
    b.forward(torch.zeros_like(x), b.plan(one, 3, 1))
    for t in range(steps):
        x.copy_(tokens[t])
        graph.replay()
        junk = [torch.full((n,), 7, dtype=torch.int32, device=DEV) for n in (3, 3, 200)]  # takes what is free
        plan = b.plan(one, 3, 1)
        want = b.forward(tokens[t], plan)
        b.commit(plan)
        torch.cuda.synchronize()
        assert torch.equal(y, want), t
        del junk
    assert a.held.tolist() == [n + steps for n in lengths] == b.held.tolist()
    assert a.spare.tolist() == b.spare.tolist() and torch.equal(a.table, b.table)
