"""The rest of a decoder layer that reads images, video or speech, as cases that can be timed and checked.

Beside its quantized linears, its cache and the attention over it (`perf/operators.py`), such a layer has:

- `norm`: the sum of a linear's output and the residual stream, its RMS norm, and that in 8 bits with a
  scale a row, as the next linear reads it (int8 rows rotated by the block Hadamard of 256, or E4M3 rows);
  the codes are read back into 16 bits, a pass of its own;
- `rope`: queries and keys normed by head and rotated to positions on several axes (time, height, width),
  each axis turning its share of a head's pairs;
- `cross`: the decoder's rows, those of one request after another, attending to an encoder's states of
  another length, from one token a request to whole videos over a text.

Activations are normal with a few louder channels, as a projection's outputs are; queries and keys are
views of the projections' buffers. How many rows and states a request has follows from the case alone.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "cozy-runtime_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_CODE = {"int8": 127.0, "fp8": 448.0}
SCALE_FLOOR = 1e-12
EPS = 1e-6
#: No drawn case costs more than the largest listed ones: elements of a norm or a rotation, an attention's
#: operations, its query-state pairs in one rectangle a request, and the states it reads.
MOST_NORM, MOST_ROPE = 6001 * 4096, 8191 * 40 * 128
MOST_WORK, MOST_PAIRS, MOST_STATES = 220e9, 5 * 32 * 800 * 6404, 40_000 * 1024


def _norm_case(rows, width, codes, dtype="bf16") -> dict:
    return {"op": "norm", "rows": rows, "width": width, "codes": codes, "dtype": dtype}


def _rope_case(tokens, heads, kv_heads, width, sections, cycled=False, interleaved=False, dtype="bf16") -> dict:
    return {"op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "width": width,
            "sections": sections, "cycled": cycled, "interleaved": interleaved, "dtype": dtype}  # fmt: skip


def _cross_case(requests, tokens, states, heads, kv_heads, width, masked=False, dtype="bf16") -> dict:
    return {"op": "cross", "requests": requests, "tokens": tokens, "states": states, "heads": heads,
            "kv_heads": kv_heads, "width": width, "masked": masked, "dtype": dtype}  # fmt: skip


def listed() -> list[dict]:
    return [
        # One user's chat, one token: hardly any work, all latency.
        dict(_norm_case(1, 4096, "int8"), name="norm_chat_1"),
        # A decode step of a small server.
        dict(_norm_case(48, 5120, "fp8"), name="norm_decode_48"),
        # A prompt, an odd number of tokens.
        dict(_norm_case(6001, 4096, "int8"), name="norm_prompt_6001"),
        # An image transformer's joint sequence in wide rows, fp16.
        dict(_norm_case(1531, 12288, "fp8", "fp16"), name="norm_wide_1531"),
        # A decode step's queries and keys, views of one QKV buffer; three axes in runs of pairs.
        dict(_rope_case(24, 32, 8, 128, "16,24,24"), name="rope_decode_24"),
        # A prompt of text and video frames, the axes' pairs taken in turns.
        dict(_rope_case(8191, 32, 8, 128, "24,20,20", True), name="rope_video_8191"),
        # An image transformer's joint sequence: as many key heads, adjacent pairs, runs of odd length, fp16.
        dict(_rope_case(4173, 20, 20, 64, "6,13,13", False, True, "fp16"), name="rope_image_4173"),
        # One speaker's next token over 1500 frames: hardly any work, all latency.
        dict(_cross_case(1, 1, 1500, 20, 20, 64, False, "fp16"), name="cross_speech_1500"),
        # A decode step of 24 requests, each over its own image's states.
        dict(_cross_case(24, 24, 1601, 32, 8, 128), name="cross_decode_24"),
        # Prompts of five requests over up to four image tiles each, some of whose states are hidden.
        dict(_cross_case(5, 2311, 6404, 32, 8, 128, True), name="cross_prompt_2311"),
        # Two videos' tokens over their texts.
        dict(_cross_case(2, 18001, 512, 24, 24, 128), name="cross_video_18001"),
        # A question of 301 tokens over a long recording, fp16.
        dict(_cross_case(1, 301, 30001, 28, 4, 128, False, "fp16"), name="cross_long_30001"),
    ]  # fmt: skip


def _log(rng, low: float, high: float) -> int:
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


HEADS = ((32, 8, 128), (16, 16, 64), (28, 4, 128), (64, 8, 128), (16, 2, 256), (12, 12, 128), (8, 1, 64), (20, 20, 64),
         (10, 10, 96), (8, 8, 80))  # fmt: skip


def draw(rng) -> dict:
    op = rng.choice(("norm", "norm", "rope", "cross", "cross", "cross"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "norm":
        codes = rng.choice(("int8", "fp8"))
        step = 256 if codes == "int8" else 16
        width = step * _log(rng, 1024 / step, 16384 / step)
        return _norm_case(_log(rng, 1, MOST_NORM / width), width, codes, dtype)
    heads, kv_heads, width = rng.choice(HEADS)
    if op == "rope":
        pairs = rng.choice((width // 2, width // 4 // 8 * 8))
        axes = rng.choice((2, 3, 3, 4))
        cycled = rng.random() < 0.4
        later = [rng.randint(1, pairs // axes) for _ in range(axes - 1)]
        sections = ",".join(map(str, [pairs - sum(later), *later]))
        tokens = _log(rng, 1, MOST_ROPE // ((heads + kv_heads) * width))
        return _rope_case(tokens, heads, kv_heads, width, sections, cycled, rng.random() < 0.4, dtype)
    requests = _log(rng, 1, 48)
    states = _log(rng, 8, min(40_000, MOST_STATES / (requests * kv_heads * width)))
    tokens = requests * rng.choice((1, 1, 5)) if rng.random() < 0.5 else requests + _log(rng, 16, 18000)
    masked = rng.random() < 0.4
    while True:
        case = _cross_case(requests, tokens, states, heads, kv_heads, width, masked, dtype)
        pairs = requests * max(_counts(case)[0]) * states * heads
        if (pairs <= MOST_PAIRS and work(case)["flops"] <= MOST_WORK) or tokens <= requests:
            return case
        tokens = max(requests, tokens * 2 // 3)


def _counts(case) -> tuple[list[int], list[int]]:
    """Rows that each request brings and states that it has: spread by the golden ratio. As many rows
    each where they divide evenly, else uneven shares; from a quarter of the longest states to all of
    them, the first the longest; one request in nine has none (a text without an image)."""
    requests, tokens = case["requests"], case["tokens"]
    golden = (math.sqrt(5) - 1) / 2
    spread = [(1 - i * golden) % 1 if i else 1.0 for i in range(requests)]
    lengths = [0 if i % 9 == 8 else max(1, round(case["states"] * (0.25 + 0.75 * s))) for i, s in enumerate(spread)]
    if tokens % requests == 0:
        return [tokens // requests] * requests, lengths
    share = [0.5 + spread[(i + 1) % requests] for i in range(requests)]
    rows = [1 + int((tokens - requests) * s / sum(share)) for s in share]
    rows[-1] += tokens - sum(rows)
    return rows, lengths


# ------------------------------------------------------------------------------ inputs


def _rows(gen, shape, dtype):
    """`shape` with a sixteenth of the last axes' channels four times louder."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= 1 + 3 * (torch.rand(shape[1:], generator=gen, device="cuda") < 1 / 16)
    return x.to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case: dict, seed: int):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = SimpleNamespace(**case)
    s.dtype = DTYPES[s.dtype]
    if s.op == "norm":
        s.x = _rows(gen, (s.rows, s.width), s.dtype)
        # The residual stream is larger than what one layer adds to it.
        s.residual = (4 * _rows(gen, (s.rows, s.width), torch.float32)).to(s.dtype)
        s.gain = (1 + 0.1 * torch.randn(s.width, generator=gen, device="cuda")).to(s.dtype)
        return s
    if s.op == "rope":
        s.sections = tuple(map(int, s.sections.split(",")))
        buffer = _rows(gen, (s.tokens, s.heads + 2 * s.kv_heads, s.width), s.dtype)
        s.q, s.k = buffer[:, : s.heads], buffer[:, s.heads : s.heads + s.kv_heads]
        s.q_gain, s.k_gain = (1 + 0.1 * torch.randn(2, s.width, generator=gen, device="cuda")).to(s.dtype).unbind(0)
        pairs, rows = sum(s.sections), s.tokens + 500
        angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs
        )
        s.cos, s.sin = angle.cos().float(), angle.sin().float()
        # An eighth of the tokens are text, all axes alike; the others frames of a square, each axis its own.
        text = s.tokens // 8
        side = max(1, math.isqrt(s.tokens) // 3)
        at = torch.arange(s.tokens, device="cuda")
        i = (at - text).clamp(min=0)
        grid = torch.stack((i // (side * side), i // side % side, i % side, i % 7))[: len(s.sections)]
        first = int(torch.randint(0, 400, (1,), generator=gen, device="cuda"))
        s.positions = (first + torch.where(at < text, at, text + grid)).to(torch.int32).contiguous()
        return s
    rows, lengths = _counts(case)
    s.most = max(rows)
    s.starts = _ints([sum(rows[:i]) for i in range(s.requests + 1)])
    s.lengths = _ints(lengths)
    s.q = _rows(gen, (s.tokens, s.heads, s.width), s.dtype)
    # The encoder's keys and values, one projection's buffer, padded to the longest.
    buffer = _rows(gen, (s.requests, s.states, 2 * s.kv_heads, s.width), s.dtype)
    s.k, s.v = buffer[:, :, : s.kv_heads], buffer[:, :, s.kv_heads :]
    s.mask = None
    if s.masked:  # runs of 25 states are hidden, a fifth of them
        runs = torch.rand(s.requests, -(-s.states // 25), generator=gen, device="cuda") >= 0.2
        s.mask = runs.repeat_interleave(25, 1)[:, : s.states].contiguous()
    return s


# ------------------------------------------------------------------------------ one pass


def run(s):
    if not own:
        return {"norm": _plain_norm, "rope": _plain_rope, "cross": _plain_cross}[s.op](s)
    if s.op == "norm":
        from cozyq import norms, operands, prebuilt

        provider = operands.INT8_CONVROT if s.codes == "int8" else operands.ROWWISE_FP8
        operand, total = norms.add_rms(torch, s.x, s.residual, s.gain, provider=provider, eps=EPS)
        # Read back as the numbers the codes stand for: a scale a row, in the rows' type.
        values = torch.empty_like(s.x)
        prebuilt.library(s.x.get_device()).decode_table(
            0 if s.codes == "int8" else 1, operand.payload, operand.scale, 0, values, s.rows, s.width, grid=1
        )
        return total, values
    if s.op == "rope":
        from cozyq import heads

        return heads.norm_rope(torch, s.q, s.k, s.q_gain, s.k_gain, s.cos, s.sin, s.positions, eps=EPS,
                               interleaved=s.interleaved, sections=s.sections, cycled=s.cycled)  # fmt: skip
    from cozyq import attention

    return attention.cross(torch, s.q, s.k, s.v, starts=s.starts, lengths=s.lengths, mask=s.mask, most=s.most)


def _hadamard(dtype):
    """The 256-point Hadamard matrix of the int8 rows, of norm 1."""
    h = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], dtype=dtype, device="cuda") / 2
    two = torch.kron(h, h)
    return torch.kron(two, two)


def _plain_norm(s):
    total = (s.x.float() + s.residual.float()).to(s.dtype)
    # The norm is that of the stream as it is stored: what any later reader of it sees.
    t = total.float()
    n = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * s.gain.float()
    if s.codes == "int8":
        n = (n.view(-1, 256) @ _hadamard(torch.float32)).view(s.rows, s.width)
    most = MOST_CODE[s.codes]
    scale = (n.abs().amax(-1, keepdim=True) / most).clamp(min=SCALE_FLOOR)
    q = (n / scale).clamp(-most, most)
    q = q.round() if s.codes == "int8" else q.to(torch.float8_e4m3fn).float()
    return total, (q * scale).to(s.dtype)


def _axis_of_pairs(sections, cycled):
    """[pairs]: the axis that each pair turns on. In runs of `sections` pairs; or, `cycled`, axis a > 0
    has pairs a, a + A, a + 2A, ... of A axes, `sections[a]` of them, and axis 0 the rest."""
    counts = torch.tensor(sections, device="cuda")
    axes, pairs = len(sections), sum(sections)
    if not cycled:
        return torch.repeat_interleave(torch.arange(axes, device="cuda"), counts, output_size=pairs)
    i = torch.arange(pairs, device="cuda")
    return torch.where(i // axes < counts[i % axes], i % axes, 0)


def _plain_rope(s):
    axis = _axis_of_pairs(s.sections, s.cycled)
    row = s.positions.long()[axis].T  # [tokens, pairs]
    cos, sin = s.cos.gather(0, row)[:, None], s.sin.gather(0, row)[:, None]
    half = sum(s.sections)

    def one(x, gain):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.float()
        turn, rest = x[..., : 2 * half], x[..., 2 * half :]
        if s.interleaved:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = turn[..., :half], turn[..., half:]
            turn = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turn, rest), -1).to(s.dtype)

    return one(s.q, s.q_gain), one(s.k, s.k_gain)


def _plain_cross(s):
    """Every request's rows against its states in one padded rectangle, masked, in float32."""
    requests, group = s.requests, s.heads // s.kv_heads
    k = s.k.float().transpose(1, 2).reshape(requests * s.kv_heads, s.states, s.width)
    v = s.v.float().transpose(1, 2).reshape(requests * s.kv_heads, s.states, s.width)
    starts = s.starts.long()
    i = torch.arange(s.most, device="cuda")
    token = (starts[:-1, None] + i).clamp(max=s.tokens - 1)
    q = s.q.float()[token].view(requests, s.most, s.kv_heads, group, s.width).transpose(1, 2)
    score = torch.bmm(q.reshape(requests * s.kv_heads, s.most * group, s.width), k.transpose(1, 2).contiguous())
    score = score.view(requests, s.kv_heads, s.most * group, s.states).mul_(s.width**-0.5)
    seen = torch.arange(s.states, device="cuda") < s.lengths[:, None]
    if s.mask is not None:
        seen &= s.mask
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.bmm(score.view(requests * s.kv_heads, s.most * group, s.states), v)
    out = out.view(requests, s.kv_heads, s.most, group, s.width)
    out = out / torch.where(total > 0, total, 1.0).view(requests, s.kv_heads, s.most, group, 1)
    out = out.transpose(1, 2).reshape(requests * s.most, s.heads, s.width)
    row = torch.arange(s.tokens, device="cuda")
    request = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return out[request * s.most + row - starts[request]].to(s.dtype)


# ------------------------------------------------------------------------------ work


def work(case: dict) -> dict:
    """Each input once, each output once."""
    c = SimpleNamespace(**case)
    if c.op == "norm":
        # x, the residual and their sum in 16 bits and the codes; then the codes and what they stand for.
        values, rotation = c.rows * c.width, 8 if c.codes == "int8" else 0
        return {"bytes": (7 + 3) * values + 8 * c.rows + 2 * c.width, "flops": (8 + rotation) * values}
    if c.op == "rope":
        values = c.tokens * (c.heads + c.kv_heads) * c.width
        axes = c.sections.count(",") + 1
        return {"bytes": 4 * values + 4 * axes * c.tokens, "flops": 7 * values}
    rows, lengths = _counts(case)
    read = 2 * 2 * sum(n for r, n in zip(rows, lengths) if r) * c.kv_heads * c.width
    pairs = sum(r * n for r, n in zip(rows, lengths))
    masks = c.requests * c.states if c.masked else 0
    return {"bytes": read + masks + 4 * c.tokens * c.heads * c.width, "flops": 4 * pairs * c.heads * c.width}


# ------------------------------------------------------------------------------ 64 bits


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "cross": _exact_cross}[s.op](s)


def _exact_norm(s):
    # The sum of two 16-bit numbers of like size is exact in 64 bits, and rounded to the stream's type once.
    total = (s.x.double() + s.residual.double()).to(s.dtype)
    t = total.double()
    n = s.gain.double() * t / (t.square().sum(-1, keepdim=True) / s.width + EPS).sqrt()
    if s.codes == "int8":
        turned = n.view(s.rows, -1, 4, 4, 4, 4)
        for axis in (2, 3, 4, 5):
            # Each row of the 4 x 4 matrix is the four's sum with one of them twice taken away.
            turned = (turned.sum(axis, keepdim=True) - 2 * turned.flip(axis)) / 2
        n = turned.reshape(s.rows, s.width)
    most = MOST_CODE[s.codes]
    scale = (n.abs().amax(-1, keepdim=True) / most).clamp(min=SCALE_FLOOR)
    q = n / scale
    if s.codes == "int8":
        q = q.round()
    else:  # three bits of significand, steps of 2^-9 at the least
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0**-6))) - 3)
        q = (q / step).round() * step
    return total.double(), q.clamp(-most, most) * scale


def _exact_rope(s):
    """As complex numbers: each pair, after its head's norm, times the table's e^(i angle) on its axis."""
    axes, pairs = len(s.sections), sum(s.sections)
    axis = []
    for a, n in enumerate(s.sections):
        axis += [a] * n
    if s.cycled:
        axis = [0] * pairs
        for a in range(1, axes):
            axis[a : a + axes * s.sections[a] : axes] = [a] * s.sections[a]
    turn = torch.stack([torch.complex(s.cos.double(), s.sin.double())[s.positions[a].long(), i] for i, a in enumerate(axis)], 1)
    out = []
    for x, gain in ((s.q, s.q_gain), (s.k, s.k_gain)):
        x = x.double()
        x = gain.double() * x / (x.square().sum(-1, keepdim=True) / s.width + EPS).sqrt()
        head = x[..., : 2 * pairs]
        both = head.unflatten(-1, (-1, 2)) if s.interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(both.contiguous()) * turn[:, None])
        x[..., : 2 * pairs] = (turned if s.interleaved else turned.transpose(-1, -2)).flatten(-2)
        out.append(x)
    return tuple(out)


def _exact_cross(s):
    out = torch.zeros(s.tokens, s.heads, s.width, dtype=torch.float64, device="cuda")
    starts, lengths = s.starts.tolist(), s.lengths.tolist()
    group = s.heads // s.kv_heads
    for r, length in enumerate(lengths):
        first, last = starts[r], starts[r + 1]
        seen = torch.arange(length, device="cuda")
        if s.mask is not None:
            seen = seen[s.mask[r, :length]]
        if first == last or not len(seen):
            continue
        for h in range(s.heads):
            k, v = s.k[r, seen, h // group].double(), s.v[r, seen, h // group].double()
            out[first:last, h] = (s.q[first:last, h].double() @ k.T / math.sqrt(s.width)).softmax(-1) @ v
    return out
