"""GPU parity of the residual norm in 8 bits (`cozyq.norms`) and of positions on several axes
(`cozyq.heads.norm_rope(sections=)`) against `oracle/layer.py`.

Bars, by what each operator rounds:
- the sum is exact in float32 and rounded once to the rows' type: equal;
- a normed element is off by 2^-18 of itself at the most: the squares' sum in float32 in up to 32 + 6 + 16 steps of
  2^-24, halved by the root, the root and two products; the rotation's eight additions and four products a value add
  16·2^-24 of the magnitudes that it sums. The scale is off as its largest element is;
- a code is the nearest of the format to the element over the scale: half a step, 1/2 (int8) or 2^-4 of it (E4M3,
  2^-10 below its normals), beside what the element and the scale are off;
- norm_rope: as in test_gpu_kv_cache.py."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import cache as law
from oracle import layer
from test_gpu_kv_cache import DEV, check_rope, rope_inputs

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def norms():
    from cozyq import norms

    return norms


def provider(codes):
    from cozyq import operands

    return operands.INT8_CONVROT if codes is torch.int8 else operands.ROWWISE_FP8


def rows_of(shape, dtype, seed, loud=4.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    x *= 1 + 3 * (torch.rand(shape[-1], generator=gen) < 1 / 16)
    r = loud * torch.randn(shape, generator=gen)
    gain = 1 + 0.3 * torch.randn(shape[-1], generator=gen)
    return x.to(dtype).to(DEV), r.to(dtype).to(DEV), gain.to(DEV)


def check(operand, total, x, r, gain, codes, eps=1e-6):
    want, n, scale, summed = layer.add_rms(x, r, gain, codes, eps)
    assert torch.equal(total, want)
    flat = (-1, x.shape[-1])
    n, summed, scale = n.view(flat), summed.view(flat), scale.view(-1, 1)
    assert operand.payload.dtype is codes and operand.payload.shape == n.shape and operand.shape == tuple(x.shape)
    off = n.abs() * 2.0**-18 + summed * (2.0**-20 if codes is torch.int8 else 0)  # of an element
    top = off.amax(-1, keepdim=True)
    got = operand.scale.double().view(-1, 1)
    assert operand.scale.shape == (n.shape[0],)
    assert ((got - scale).abs() <= top / layer.MOST[codes] + scale * 2.0**-22).all()
    code, value = operand.payload.double(), n / got
    half = torch.full_like(value, 0.5) if codes is torch.int8 else (value.abs() * 2.0**-4).clamp(min=2.0**-10)
    bar = half * (1 + 2.0**-20) + off / got + value.abs() * 2.0**-22
    error = (code - value.clamp(-layer.MOST[codes], layer.MOST[codes])).abs()
    assert (error <= bar).all(), float((error / bar).max())


WIDTHS = {torch.int8: [256, 512, 1280, 4096, 5120, 16384, 16640, 32768], E4M3: [16, 48, 1040, 4096, 12288, 16384, 16400, 32768]}


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("codes,width", [(c, w) for c in WIDTHS for w in WIDTHS[c]], ids=lambda v: str(v).split(".")[-1])
def test_add_rms(norms, codes, width, dtype):
    for rows in (1, 3, 130):
        x, r, gain = rows_of((rows, width), dtype, rows + width)
        for g in (gain, gain.to(dtype)):
            operand, total = norms.add_rms(torch, x, r, g, provider=provider(codes))
            check(operand, total, x, r, g, codes)


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
def test_add_rms_parts_left_out_and_shapes(norms, codes):
    """No residual, no gain, leading axes, rows of a wider buffer, no rows."""
    how = dict(provider=provider(codes))
    x, r, gain = rows_of((2, 5, 512), BF16, 7)
    operand, total = norms.add_rms(torch, x, None, gain, **how)
    assert total is x
    check(operand, total, x, None, gain, codes)
    operand, total = norms.add_rms(torch, x, r, None, eps=0.5, **how)
    check(operand, total, x, r, None, codes, 0.5)
    wide = torch.randn(6, 1030, device=DEV).to(BF16)
    for view in (wide[:, :512], wide[:, 3:515], wide[::2, 512:1024]):
        other = r.view(-1, 512)[: view.shape[0]]
        operand, total = norms.add_rms(torch, view, other, gain, **how)
        check(operand, total, view, other, gain, codes)
        operand, total = norms.add_rms(torch, other, view, gain, **how)
        check(operand, total, other, view, gain, codes)
    operand, total = norms.add_rms(torch, x[:0], r[:0], gain, **how)
    assert operand.payload.shape == (0, 512) and operand.scale.shape == (0,) and total.shape == (0, 5, 512)


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
@pytest.mark.parametrize("width", [512, 20480])
def test_add_rms_in_place(norms, codes, width):
    x, r, gain = rows_of((37, width), BF16, 8)
    want, sums = norms.add_rms(torch, x, r, gain, provider=provider(codes))
    for into in ("residual", "x", "new"):
        a, b = x.clone(), r.clone()
        out = {"residual": b, "x": a, "new": torch.empty_like(x)}[into]
        operand, total = norms.add_rms(torch, a, b, gain, provider=provider(codes), out=out)
        assert total is out and torch.equal(total, sums)
        assert torch.equal(operand.payload.view(torch.int8), want.payload.view(torch.int8)) and torch.equal(operand.scale, want.scale)
        assert into == "x" or torch.equal(a, x)
        assert into == "residual" or torch.equal(b, r)


@pytest.mark.parametrize("codes", [torch.int8, E4M3], ids=["int8", "fp8"])
def test_add_rms_of_zeros_tiny_huge_and_not_finite_rows(norms, codes):
    x = torch.zeros(9, 512, dtype=BF16)
    x[1], x[2], x[3] = 1e-30, 1.0, 2.0**60
    x[4, 7], x[5, 500], x[6, 3] = math.inf, -math.inf, math.nan
    x[7, 0] = 2.0**-130  # a subnormal among zeros
    x[8] = 2.0**100
    r = torch.zeros_like(x)
    x, r = x.to(DEV), r.to(DEV)
    operand, total = norms.add_rms(torch, x, r, None, provider=provider(codes))
    assert torch.equal(total.view(torch.int16), (x + r).view(torch.int16))
    keep = [0, 1, 2, 3, 8]
    part = type(operand)(operand.payload[keep], operand.scale[keep], (5, 512), operand.provider)
    check(part, total[keep], x[keep], r[keep], None, codes)
    assert (operand.payload[0].float() == 0).all() and operand.scale[0].item() == pytest.approx(1e-12)
    assert operand.scale[4:7].isnan().all() and operand.scale[7].isfinite()


def test_add_rms_refusals(norms):
    x, r, gain = rows_of((4, 512), BF16, 9)
    good = dict(x=x, residual=r, gain=gain, provider=provider(torch.int8), eps=1e-6, out=None)
    buffer = torch.zeros(6, 512, dtype=BF16, device=DEV)
    for bad in (dict(x=x.float()), dict(x=x.cpu()), dict(residual=r.half()), dict(residual=r[:3]), dict(residual=r.cpu()),
                dict(x=x[:, :384], residual=r[:, :384], gain=gain[:384]), dict(x=x[:, :0], residual=r[:, :0], gain=None),
                dict(gain=gain[:256]), dict(gain=gain.half()), dict(gain=gain.cpu()), dict(gain=gain.double()),
                dict(gain=torch.zeros(513, device=DEV)[1:]), dict(provider="cozy.mxfp8.native-leaf/2"), dict(eps=0.0), dict(eps=-1.0),
                dict(out=torch.empty_like(x, dtype=FP16)), dict(out=x[:3]), dict(out=x.cpu()), dict(out=torch.empty(512, 4, dtype=BF16, device=DEV).T),
                dict(residual=None, out=r), dict(x=buffer[:4], out=buffer[1:5]), dict(residual=buffer[2:], out=buffer[:4]),
                dict(x=x[0, 0], residual=r[0, 0], gain=None)):  # fmt: skip
        with pytest.raises(ValueError):
            norms.add_rms(torch, **(good | bad))


def test_add_rms_past_32_bit_offsets(norms):
    """Rows whose elements pass 2^31, the last ones against the same rows alone."""
    rows, width = 66000, 32768
    x = torch.zeros(rows, width, dtype=BF16, device=DEV)
    small, r, gain = rows_of((3, width), BF16, 10)
    x[-3:] = small
    stream = torch.zeros_like(x)
    stream[-3:] = r
    for codes in (torch.int8, E4M3):
        want, sums = norms.add_rms(torch, small, r, gain, provider=provider(codes))
        operand, total = norms.add_rms(torch, x, stream, gain, provider=provider(codes))
        assert torch.equal(total[-3:], sums) and torch.equal(operand.scale[-3:], want.scale)
        assert torch.equal(operand.payload[-3:].view(torch.int8), want.payload.view(torch.int8))
        assert not operand.payload[0].float().any()  # zeros of either sign, as the gain is
        del operand, total


def test_add_rms_in_a_graph_and_on_another_stream(norms):
    x, r, gain = rows_of((70, 1024), FP16, 11)
    how = dict(provider=provider(torch.int8))
    first, _ = norms.add_rms(torch, x, r, gain, **how)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other, _ = norms.add_rms(torch, x, r, gain, **how)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other.payload, first.payload) and torch.equal(other.scale, first.scale)
    torch.cuda.synchronize()
    state = r.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = norms.add_rms(torch, x, state, gain, out=state, **how)
    want = r.clone()
    for _ in range(3):
        operand, _ = norms.add_rms(torch, x, want, gain, out=want, **how)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(state, want) and torch.equal(got.payload, operand.payload) and torch.equal(got.scale, operand.scale)


def test_add_rms_feeds_the_linears(norms):
    """The operand through int8.convrot's and fp8.rowwise's GEMMs, as the linear of the normed rows in 64 bits within
    the codes' own rounding: half a step of the largest over 127 an element (int8), 2^-4 of each (E4M3), their
    magnitudes added up over K."""
    from cozyq import fp8_linear, int8_linear
    from oracle import laws

    gen = torch.Generator().manual_seed(12)
    w = torch.randn(64, 512, generator=gen) * 0.05
    x, r, gain = rows_of((33, 512), BF16, 13)
    for codes, op, made in ((torch.int8, int8_linear, laws.int8_weight_rotated(w, 256)), (E4M3, fp8_linear, laws.fp8_weight(w))):
        operand, _ = norms.add_rms(torch, x, r, gain, provider=provider(codes))
        y = op.gemm(torch, operand, made[0].to(DEV), made[1].to(DEV).view(-1), None, BF16).double()
        _, n, scale, _ = layer.add_rms(x, r, gain, codes, 1e-6)
        weight = made[0].double().to(DEV) * made[1].double().to(DEV).view(-1, 1)
        size = weight.abs().sum(-1)[None] * scale / 2 if codes is torch.int8 else (n.abs() @ weight.abs().T) * 2.0**-4
        assert ((y - n @ weight.T).abs() <= 1.01 * size + 2.0**-7 * y.abs() + 1e-3).all()


# ------------------------------------------------------------------------------ axes


SHARES = [((4, 2, 2), False), ((4, 2, 2), True), ((3, 5), False), ((4, 4), True), ((2, 1, 3, 2), False), ((5, 1, 1, 1), True),
          ((0, 0, 8), False), ((8, 0, 0), True)]  # fmt: skip


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("tokens,heads,k_heads,width,rotated", [
    (1, 1, 1, 16, 16), (1, 32, 8, 128, 128), (33, 12, 12, 80, 80), (130, 3, 1, 96, 48), (19, 7, 2, 256, 256),
    (601, 6, 2, 128, 64), (5, 4, 4, 192, 160), (2900, 5, 3, 64, 64)])  # fmt: skip
def test_norm_rope_on_axes(tokens, heads, k_heads, width, rotated, interleaved, dtype):
    from cozyq import heads as ops

    qkv, cos, sin, _, gains = rope_inputs(tokens, heads, k_heads, width, rotated, dtype, tokens + width)
    on, gains = qkv.to(DEV), gains.to(dtype)
    q, k = on[:, :heads], on[:, heads : heads + k_heads]
    gen = torch.Generator().manual_seed(width)
    for shares, cycled in SHARES if tokens < 200 else SHARES[1:3]:
        many = rotated // 16
        sections = tuple(n * many for n in shares)
        if rotated > 16:  # odd counts
            sections = (sections[0] + 1, sections[1] - 1, *sections[2:]) if sections[1] else sections
        positions = torch.randint(-3, cos.shape[0] + 3, (len(sections), tokens), generator=gen, dtype=torch.int32)
        got = ops.norm_rope(torch, q, k, gains[0].contiguous().to(DEV), gains[1].contiguous().to(DEV), cos.to(DEV), sin.to(DEV),
                            positions.to(DEV), eps=1e-5, interleaved=interleaved, sections=sections, cycled=cycled)  # fmt: skip
        turn = layer.tables(cos, sin, positions, sections, cycled)
        for part, x, gain in zip(got, (q, k), gains):
            check_rope(part, *law.norm_rope(x.cpu(), gain, *turn, None, 1e-5, interleaved), dtype)


def test_norm_rope_on_axes_that_agree_is_one_axis_bit_for_bit():
    from cozyq import heads as ops

    qkv, cos, sin, positions, _ = (x.to(DEV) for x in rope_inputs(300, 6, 2, 128, 128, BF16, 21))
    one = ops.norm_rope(torch, qkv[:, :6], qkv[:, 6:8], None, None, cos, sin, positions)
    for sections, cycled in (((20, 20, 24), False), ((24, 20, 20), True)):
        three = positions.expand(3, -1).contiguous()
        got = ops.norm_rope(torch, qkv[:, :6], qkv[:, 6:8], None, None, cos, sin, three, sections=sections, cycled=cycled)
        assert torch.equal(got[0], one[0]) and torch.equal(got[1], one[1])


def test_norm_rope_on_axes_without_norm_or_keys_and_in_a_graph():
    from cozyq import heads as ops

    qkv, cos, sin, _, _ = rope_inputs(40, 4, 1, 64, 64, FP16, 22)
    q, positions = qkv[:, :4].to(DEV), torch.randint(0, 80, (2, 40), dtype=torch.int32, generator=torch.Generator().manual_seed(1))
    how = dict(eps=None, sections=(15, 17))
    at = positions.to(DEV)
    got, none = ops.norm_rope(torch, q, None, None, None, cos.to(DEV), sin.to(DEV), at, **how)
    assert none is None
    check_rope(got, *law.norm_rope(q.cpu(), None, *layer.tables(cos, sin, positions, (15, 17), False), None, None, False), FP16)
    assert ops.norm_rope(torch, q[:0], None, None, None, cos.to(DEV), sin.to(DEV), at[:, :0].contiguous(), **how)[0].shape == (0, 4, 64)
    c, s = cos.to(DEV), sin.to(DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = ops.norm_rope(torch, q, None, None, None, c, s, at, **how)
    for _ in range(3):
        at.add_(1)
        want, _ = ops.norm_rope(torch, q, None, None, None, c, s, at, **how)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_norm_rope_on_axes_refusals():
    from cozyq import heads as ops

    qkv, cos, sin, _, _ = (x.to(DEV) for x in rope_inputs(4, 2, 2, 64, 64, BF16, 23))
    at = torch.zeros(3, 4, dtype=torch.int32, device=DEV)
    good = dict(positions=at, sections=(8, 12, 12), cycled=False, cos=cos, sin=sin)
    for bad in (dict(sections=(8, 12, 11)), dict(sections=(32,)), dict(sections=(8, 6, 6, 6, 6)), dict(sections=(8, 30, -6)),
                dict(sections=()), dict(sections=(2, 15, 15), cycled=True), dict(sections=None, cycled=True),
                dict(sections=None), dict(positions=None), dict(positions=at[:2]), dict(positions=at.long()), dict(positions=at[0]),
                dict(positions=at[:, :3]), dict(positions=torch.zeros(4, 3, dtype=torch.int32, device=DEV).T), dict(positions=at.cpu()),
                dict(cos=None, sin=None)):  # fmt: skip
        a = good | bad
        with pytest.raises(ValueError):
            ops.norm_rope(torch, qkv[:, :2], qkv[:, 2:4], None, None, a["cos"], a["sin"], a["positions"], sections=a["sections"],
                          cycled=a["cycled"])  # fmt: skip
