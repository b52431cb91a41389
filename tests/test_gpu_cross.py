"""GPU parity of attention to an encoder's states (`cozyq.attention.cross`) against `oracle/layer.py`.

Bars, by what the operator rounds: u·|y| for the output's one rounding, u = 2^-8 (bf16) or 2^-11 (fp16); of Σ p·|v|
the weights' rounding, another u, and what the scores are off in float32: (D + 8)·2^-24 of Σ|q|·|k|·scale, twice as a
weight and its denominator are off by it, and 2^-20 for the sums; and in fp16, whose weights end at 2^-25 with the
largest at 2^6 at the least, 2^-31 of Σ|v|."""

from __future__ import annotations

import math
import random

import pytest
import torch

from oracle import layer
from test_gpu_kv_cache import DEV, UNIT, ints

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def attention():
    from cozyq import attention

    return attention


def inputs(tokens, requests, states, heads, kv_heads, width, dtype, seed):
    """q a view of a wider buffer, k and v of one projection's, a sixteenth of the channels four times louder."""
    gen = torch.Generator(DEV).manual_seed(seed)

    def rows(*shape):
        x = torch.randn(*shape, generator=gen, device=DEV)
        x *= 1 + 3 * (torch.rand(shape[-2:], generator=gen, device=DEV) < 1 / 16)
        return x.to(dtype)

    q = rows(tokens, heads + 3, width)[:, 2 : heads + 2]
    kv = rows(requests, states, 2 * kv_heads, width)
    return q, kv[:, :, :kv_heads], kv[:, :, kv_heads:]


def counts(rows):
    return ints([sum(rows[:i]) for i in range(len(rows) + 1)])


def bar(q, k, v, want, size, scale=None):
    """The module's bars [tokens, heads, 1 or D]; every state is taken for the largest, seen or not."""
    if not k.shape[1]:
        return torch.zeros_like(want)
    dtype, width = q.dtype, q.shape[-1]
    scale = width**-0.5 if scale is None else abs(scale)
    group = q.shape[1] // k.shape[2]
    clean = k.double().nan_to_num(0.0, 0.0, 0.0)
    most = clean.abs().amax((0, 1)).repeat_interleave(group, 0)  # [heads, D]
    off = 2 * (width + 8) * 2.0**-24 * scale * (q.double().abs() * most).sum(-1, keepdim=True) + 2.0**-20
    tail = 0.0
    if dtype is FP16:
        tail = 2.0**-31 * v.double().nan_to_num(0.0, 0.0, 0.0).abs().sum(1).amax(0).repeat_interleave(group, 0)
    return UNIT[dtype] * want.abs() + (UNIT[dtype] + off) * size + tail + (2.0**-25 if dtype is FP16 else 2.0**-130)


def check(got, q, k, v, starts, lengths, mask=None, scale=None):
    each = q.shape[0] // k.shape[0]
    starts = [each * r for r in range(k.shape[0] + 1)] if starts is None else starts.tolist()
    lengths = [k.shape[1]] * k.shape[0] if lengths is None else lengths.tolist()
    want, size = layer.cross(q, k, v, starts, lengths, mask, scale)
    error = (got.double() - want).abs()
    limit = bar(q, k, v, want, size, scale)
    assert got.dtype is q.dtype and got.is_contiguous() and got.shape == q.shape
    assert (error <= limit).all(), float((error / limit.clamp(min=1e-300)).max())


HEADS = [(4, 4, 64), (8, 2, 128), (7, 1, 64), (2, 2, 256), (6, 3, 80), (4, 2, 96), (3, 3, 8), (4, 4, 40), (2, 1, 200), (5, 5, 128)]


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,width", HEADS)
def test_cross(attention, heads, kv_heads, width, dtype):
    """From one row a request to a few hundred over states of every kind of length."""
    for rows, states, lengths in (([1], 1, [1]), ([1, 1, 1], 65, [65, 1, 64]), ([3, 0, 1, 40], 130, [128, 5, 130, 0]),
                                  ([300, 17], 77, [77, 33]), ([33], 700, [700]), ([2, 5], 1500, [1500, 1031])):  # fmt: skip
        q, k, v = inputs(sum(rows), len(rows), states, heads, kv_heads, width, dtype, states + width)
        starts, n = counts(rows), ints(lengths)
        got = attention.cross(torch, q, k, v, starts=starts, lengths=n, most=max(rows))
        check(got, q, k, v, starts, n)


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,width", [(4, 1, 128), (3, 3, 64), (2, 2, 256), (4, 2, 72)])
def test_cross_masked(attention, heads, kv_heads, width, dtype):
    """Masks of single states, of runs, of whole steps, and one that leaves nothing."""
    for rows, states in (([1, 1, 1, 1, 1], 200), ([70, 1, 2, 300, 9], 333), ([1, 1, 1, 1, 1], 2100)):
        q, k, v = inputs(sum(rows), 5, states, heads, kv_heads, width, dtype, states)
        gen = torch.Generator(DEV).manual_seed(states)
        mask = torch.rand(5, states, generator=gen, device=DEV) < 0.5
        mask[1] = True
        mask[2, :128] = False
        mask[3] = False
        mask[4, 1:] = False
        starts, n = counts(rows), ints([states, states - 1, states, states, states])
        got = attention.cross(torch, q, k, v, starts=starts, lengths=n, mask=mask, most=max(rows))
        check(got, q, k, v, starts, n, mask)
        assert not got[int(starts[3]) : int(starts[4])].any()
        wide = torch.zeros(5, states + 9, dtype=torch.bool, device=DEV)
        wide[:, 3 : states + 3] = mask
        assert torch.equal(attention.cross(torch, q, k, v, starts=starts, lengths=n, mask=wide[:, 3 : states + 3], most=max(rows)), got)


@pytest.mark.parametrize("width", [64, 128, 256, 88])
@pytest.mark.parametrize("rows", [[1, 1, 1], [200, 3, 40]], ids=["few", "many"])
def test_cross_what_is_not_seen_reaches_no_result(attention, rows, width):
    """NaN and infinities past the lengths and where the mask hides, and the type's lowest and largest numbers."""
    states = 450
    q, k, v = inputs(sum(rows), 3, states, 4, 2, width, FP16, width)
    mask = torch.rand(3, states, generator=torch.Generator(DEV).manual_seed(1), device=DEV) < 0.7
    starts, n = counts(rows), ints([450, 130, 1])
    mask[2, 0] = True
    want = attention.cross(torch, q, k, v, starts=starts, lengths=n, mask=mask, most=max(rows))
    check(want, q, k, v, starts, n, mask)
    hidden = ~mask | (torch.arange(states, device=DEV) >= n[:, None])
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(FP16).min, torch.finfo(FP16).max):
        k2, v2 = k.clone(), v.clone()
        k2[hidden], v2[hidden] = bad, bad
        got = attention.cross(torch, q, k2, v2, starts=starts, lengths=n, mask=mask, most=max(rows))
        assert torch.equal(got, want), bad


@pytest.mark.parametrize("rows", [[1, 1, 1], [200, 3, 40]], ids=["few", "many"])
def test_cross_not_finite_states_reach_the_rows_that_see_them(attention, rows):
    states = 300
    q, k, v = inputs(sum(rows), 3, states, 4, 2, 64, BF16, 5)
    starts, n = counts(rows), ints([300, 200, 100])
    clean = attention.cross(torch, q, k, v, starts=starts, lengths=n, most=max(rows))
    for tensor, bad in (("k", math.nan), ("v", math.nan), ("v", math.inf)):
        k2, v2 = k.clone(), v.clone()
        (k2 if tensor == "k" else v2)[1, 77, 1, 3] = bad
        got = attention.cross(torch, q, k2, v2, starts=starts, lengths=n, most=max(rows))
        a, b = rows[0], rows[0] + rows[1]
        assert torch.equal(got[:a], clean[:a]) and torch.equal(got[b:], clean[b:])
        assert torch.equal(got[a:b, :2], clean[a:b, :2])
        part = got[a:b, 2:] if tensor == "k" else got[a:b, 2:, 3]
        assert (~part.isfinite()).all()
    # Scores of plus infinity, and of nothing but minus infinity, are no softmax: NaN.
    q2 = q.abs() + 0.01
    for fill, lone in ((-math.inf, False), (math.inf, True)):
        k2 = k.clone()
        if lone:
            k2[0, 299] = fill
        else:
            k2[0] = fill
        got = attention.cross(torch, q2, k2, v, starts=starts, lengths=n, most=max(rows))
        assert got[: rows[0]].isnan().all() and got[rows[0] :].isfinite().all()


def test_cross_lengths_and_starts_outside_the_call(attention):
    """Lengths below 0 and past the states; rows before the first request's, after the last's and past the call's end; in
    memory that held NaN."""
    q, k, v = inputs(90, 4, 100, 2, 2, 64, BF16, 6)
    for given, meant in (([5, 6, 6, 40, 60], [5, 6, 6, 40, 60]), ([-7, 30, 31, 31, 200], [0, 30, 31, 31, 90]),
                         ([0, 0, 0, 0, 0], [0, 0, 0, 0, 0]), ([90, 90, 95, 95, 99], [90, 90, 90, 90, 90])):  # fmt: skip
        for lengths in ([100, 1, -5, 101], [2**31 - 1, 100, 0, -(2**31)]):
            how = dict(starts=ints(given), lengths=ints(lengths), most=60)
            torch.cuda.empty_cache()
            junk = [torch.full(q.shape, math.nan, dtype=BF16, device=DEV) for _ in range(4)]
            where = {x.data_ptr() for x in junk}
            del junk
            got = attention.cross(torch, q, k, v, **how)
            assert got.data_ptr() in where
            check(got, q, k, v, ints(meant), ints([min(max(n, 0), 100) for n in lengths]))
            assert not got[: meant[0]].any() and not got[meant[-1] :].any()


def test_cross_rows_as_many_for_each_request(attention):
    q, k, v = inputs(84, 7, 150, 4, 2, 128, BF16, 7)
    got = attention.cross(torch, q, k, v)
    check(got, q, k, v, None, None)
    assert torch.equal(got, attention.cross(torch, q, k, v, starts=counts([12] * 7), lengths=ints([150] * 7), most=12))
    n = ints([150, 3, 0, 64, 65, 150, 128])
    check(attention.cross(torch, q, k, v, lengths=n), q, k, v, None, n)


@pytest.mark.parametrize("states", [0, 1, 63, 64, 65, 128, 129, 4096, 16385])
def test_cross_lengths_at_the_steps_ends(attention, states):
    for rows in ([1, 2], [130, 1]):
        q, k, v = inputs(sum(rows), 2, states, 2, 1, 64, FP16, 8)
        n = ints([states, max(0, states - 1)])
        got = attention.cross(torch, q, k, v, starts=counts(rows), lengths=n, most=max(rows))
        check(got, q, k, v, counts(rows), n)


@pytest.mark.parametrize("most", [0, 1, 2, 40, 10**6])
def test_cross_results_hold_for_any_hint(attention, most):
    rows = [40, 1, 0, 7]
    q, k, v = inputs(sum(rows), 4, 900, 8, 2, 64, BF16, 9)
    n = ints([900, 850, 3, 64])
    check(attention.cross(torch, q, k, v, starts=counts(rows), lengths=n, most=most), q, k, v, counts(rows), n)


def test_cross_over_many_requests(attention):
    rng = random.Random(10)
    rows = [rng.choice((0, 1, 1, 2, 9)) for _ in range(301)]
    q, k, v = inputs(sum(rows), 301, 40, 2, 2, 64, BF16, 10)
    n = ints([rng.randint(0, 40) for _ in rows])
    for most in (0, 9):
        check(attention.cross(torch, q, k, v, starts=counts(rows), lengths=n, most=most), q, k, v, counts(rows), n)


@pytest.mark.parametrize("heads,kv_heads,width,rows,states", [
    (4, 4, 64, [3000, 1], 512), (8, 2, 128, [700, 301], 1111), (2, 1, 256, [900], 257), (64, 1, 64, [40, 3], 333),
    (28, 4, 128, [301], 9001), (3, 3, 96, [515, 515], 77)])  # fmt: skip
def test_cross_many_rows(attention, heads, kv_heads, width, rows, states):
    q, k, v = inputs(sum(rows), len(rows), states, heads, kv_heads, width, BF16, 11)
    n = ints([states, states * 2 // 3][: len(rows)])
    check(attention.cross(torch, q, k, v, starts=counts(rows), lengths=n, most=max(rows)), q, k, v, counts(rows), n)


@pytest.mark.parametrize("rows", [[2, 1], [150, 1]], ids=["few", "many"])
def test_cross_score_magnitudes(attention, rows):
    """Queries from 2^-20 to 2^10 of their usual size and scales of either sign: flat softmaxes to one state's alone."""
    q, k, v = inputs(sum(rows), 2, 400, 2, 2, 64, BF16, 12)
    n = ints([400, 399])
    for power in (-20, -3, 4, 10):
        for scale in (None, -0.05, 0.0):
            x = q * 2.0**power
            got = attention.cross(torch, x, k, v, starts=counts(rows), lengths=n, most=max(rows), scale=scale)
            check(got, x, k, v, counts(rows), n, None, scale)


def test_cross_strides(attention):
    """Heads before states, requests that share their states, padded rows, one state's stride of one."""
    gen = torch.Generator(DEV).manual_seed(13)
    q = torch.randn(6, 30, 64, generator=gen, device=DEV).to(BF16).transpose(0, 1)  # [30, 6, 64]
    kv = torch.randn(2, 3, 70, 64 + 8, generator=gen, device=DEV).to(BF16)
    k, v = kv[..., :64].transpose(1, 2), kv[..., 8:].transpose(1, 2)  # [2, 70, 3, 64]
    check(attention.cross(torch, q, k, v), q, k, v, None, None)
    one = k[:1].expand(5, -1, -1, -1), v[1:].expand(5, -1, -1, -1)
    check(attention.cross(torch, q, *one), q, *one, None, None)
    same = k[:, :1].expand(-1, 40, -1, -1), v[:, :40]
    check(attention.cross(torch, q, *same), q, *same, None, None)
    lone = torch.randn(2, 1, 3, 64, generator=gen, device=DEV).to(BF16).as_strided((2, 1, 3, 64), (192, 1, 64, 1))
    check(attention.cross(torch, q, lone, lone), q, lone, lone, None, None)


@pytest.mark.parametrize("rows", [[1, 1], [90, 200]], ids=["few", "many"])
def test_cross_past_32_bit_offsets(attention, rows):
    """Two requests' states 2^31 bytes and more from one another, and a request's last from its first."""
    buffer = torch.zeros(2, 70000, 128, 128, dtype=BF16, device=DEV)  # 4.6 GB
    gen = torch.Generator(DEV).manual_seed(14)
    for at in (7, 126):
        buffer[:, :, at] = torch.randn(2, 70000, 128, generator=gen, device=DEV).to(BF16)
    k, v = buffer[:, :, 7:8], buffer[:, :, 126:127]
    q = torch.randn(sum(rows), 2, 128, generator=gen, device=DEV).to(BF16)
    n = ints([70000, 69999])
    check(attention.cross(torch, q, k, v, starts=counts(rows), lengths=n, most=max(rows)), q, k, v, counts(rows), n)


@pytest.mark.parametrize("masked", [False, True], ids=["whole", "masked"])
@pytest.mark.parametrize("rows", [[1, 0, 2], [130, 0, 40]], ids=["few", "many"])
def test_cross_rows_of_no_request_beside_shared_out_states(attention, rows, masked):
    """Rows before the first request's and after the last's, where requests' states are shared out over workgroups."""
    q, k, v = inputs(sum(rows) + 50, 3, 2500, 4, 2, 64, BF16, 16)
    starts, n = ints([20 + sum(rows[:i]) for i in range(4)]), ints([2500, 2500, 700])
    mask = torch.rand(3, 2500, device=DEV) < 0.7 if masked else None
    torch.cuda.empty_cache()
    junk = [torch.full(q.shape, math.nan, dtype=BF16, device=DEV) for _ in range(4)]
    where = {x.data_ptr() for x in junk}
    del junk
    got = attention.cross(torch, q, k, v, starts=starts, lengths=n, mask=mask, most=max(rows))
    assert got.data_ptr() in where
    check(got, q, k, v, starts, n, mask)
    assert not got[:20].any() and not got[20 + sum(rows) :].any()


@pytest.mark.parametrize("masked", [False, True], ids=["whole", "masked"])
def test_cross_many_steps_of_one_workgroup(attention, masked):
    """Tiles enough that none's states are shared out, over more than 256 steps of 64 of them."""
    q, k, v = inputs(557, 2, 16900, 64, 64, 8, FP16, 17)
    starts, n = counts([300, 257]), ints([16900, 16385])
    mask = torch.rand(2, 16900, device=DEV) < 0.5 if masked else None
    got = attention.cross(torch, q, k, v, starts=starts, lengths=n, mask=mask, most=300)
    check(got, q, k, v, starts, n, mask)


@pytest.mark.parametrize("rows", [[1, 1, 1], [30, 1, 200]], ids=["few", "many"])
def test_cross_is_the_same_every_time_on_another_stream_and_in_a_graph(attention, rows):
    """A captured call, replayed over changing lengths, masks and rows with eager work between, equals the eager one."""
    q, k, v = inputs(sum(rows), 3, 2500, 8, 2, 64, BF16, 15)
    q = q.contiguous()
    starts, n = counts(rows), ints([2500, 5, 900])
    mask = torch.ones(3, 2500, dtype=torch.bool, device=DEV)
    how = dict(starts=starts, lengths=n, mask=mask, most=max(rows))
    first = attention.cross(torch, q, k, v, **how)
    for _ in range(4):
        assert torch.equal(attention.cross(torch, q, k, v, **how), first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = attention.cross(torch, q, k, v, **how)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, first)
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention.cross(torch, q, k, v, **how)
    with torch.cuda.graph(second):
        also = attention.cross(torch, q, k, v, **how)
    for lengths in ([2500, 5, 900], [0, 2500, 64], [1300, 0, 1], [2500, 2500, 2500]):
        n.copy_(ints(lengths))
        mask[:, 100 : 100 + lengths[0] // 2] ^= True
        q.add_(0.25)
        want = attention.cross(torch, q, k, v, **how)
        check(want, q, k, v, starts, n, mask)
        torch.cuda.synchronize()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(also, want)


def test_cross_refusals(attention):
    q, k, v = inputs(6, 3, 20, 4, 2, 64, BF16, 16)
    good = dict(q=q, k=k, v=v, starts=None, lengths=None, mask=None, most=0)
    mask = torch.ones(3, 20, dtype=torch.bool, device=DEV)
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(k=k.half()), dict(v=v.half()), dict(q=q[0]), dict(k=k[0]), dict(v=v[:, :10]),
                dict(q=q[..., :32]), dict(q=q[:, :3]), dict(k=k[:, :, :0], v=v[:, :, :0]), dict(q=q[:, :0]), dict(q=q[:5]),
                dict(q=q[..., 1:]), dict(q=q.transpose(1, 2)), dict(k=k.transpose(2, 3).contiguous().transpose(2, 3)),
                dict(k=k[:0], v=v[:0]), dict(starts=ints([0, 1, 2])), dict(starts=ints([0, 1, 2, 6]).long()), dict(starts=ints([0, 1, 2, 6]).cpu()),
                dict(lengths=ints([1, 2])), dict(lengths=torch.ones(3, device=DEV)), dict(mask=mask.to(torch.uint8)), dict(mask=mask[:, :19]),
                dict(mask=mask.T.contiguous().T), dict(mask=mask.cpu()), dict(most=-1, starts=ints([0, 1, 2, 6])), dict(q=q.cpu()),
                dict(k=k.cpu()), dict(v=v.cpu()),
                dict(q=torch.zeros(3, 4, 512, dtype=BF16, device=DEV), k=torch.zeros(3, 20, 2, 512, dtype=BF16, device=DEV), v=torch.zeros(3, 20, 2, 512, dtype=BF16, device=DEV)),
                dict(q=torch.zeros(3, 4, 12, dtype=BF16, device=DEV), k=torch.zeros(3, 20, 2, 12, dtype=BF16, device=DEV), v=torch.zeros(3, 20, 2, 12, dtype=BF16, device=DEV)),
                dict(k=torch.zeros(1, dtype=BF16, device=DEV).as_strided((3, 1, 2, 64), (0, 0, 0, 0)), v=v[:, :1])):  # fmt: skip
        a = good | bad
        with pytest.raises(ValueError):
            attention.cross(torch, a["q"], a["k"], a["v"], starts=a["starts"], lengths=a["lengths"], mask=a["mask"], most=a["most"])
    assert attention.cross(torch, q[:0], k, v).shape == (0, 4, 64)
