"""The attention side of a quantized language model's step, as cases that can be timed and checked.

The linears of such a model run on 8-bit codes; so does its cache of keys and values. A case is one
pass through one of the operators between the QKV projection and the output projection:

- `plan`: once a step, from the requests' lengths: the pages that their new tokens take from the free
  list, the block table with them, and each token's slot, position and request;
- `rope`: queries and keys as the QKV projection wrote them, each head normed and rotated to its
  token's position;
- `append`: new keys and values quantized into the cache's pages, one scale a page and head (a page
  that was begun earlier is scaled again where the new tokens need it), and those pages read back;
- `attend`: each new token's attention over its request's pages, from one token a request to whole
  prompts, causal, with a window or without.

Keys, values and queries are normal with a few louder channels, as a projection's outputs are; page
numbers come from a shuffled free list. A request's length follows from the case alone.
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
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
MOST_CODE = {"int8": 127.0, "fp8": 448.0}
SCALE_FLOOR = 1e-12
EPS = 1e-6
#: No drawn case's attention does more work than the two prompts listed, nor has more query-key pairs
#: over all heads in one rectangle a request, nor reads more cached tokens than the longest listed.
MOST_WORK, MOST_PAIRS, MOST_TOKENS = 850e9, 2 * 8192 * 8192 * 32, 160_000


def _plan_case(requests, longest, tokens, page, mode) -> dict:
    return {"op": "plan", "requests": requests, "longest": longest, "tokens": tokens, "page": page, "mode": mode}


def _rope_case(tokens, heads, kv_heads, width, rotated, interleaved=False, dtype="bf16") -> dict:
    return {"op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "width": width,
            "rotated": rotated, "interleaved": interleaved, "dtype": dtype}  # fmt: skip


def _append_case(requests, longest, tokens, mode, kv_heads, width, page, codes, dtype="bf16") -> dict:
    return {"op": "append", "requests": requests, "longest": longest, "tokens": tokens, "mode": mode,
            "kv_heads": kv_heads, "width": width, "page": page, "codes": codes, "dtype": dtype}  # fmt: skip


def _attend_case(requests, longest, tokens, mode, heads, kv_heads, width, page, codes, window=0, dtype="bf16") -> dict:
    return {"op": "attend", "requests": requests, "longest": longest, "tokens": tokens, "mode": mode,
            "heads": heads, "kv_heads": kv_heads, "width": width, "page": page, "codes": codes, "window": window,
            "dtype": dtype}  # fmt: skip


def listed() -> list[dict]:
    return [
        # A decode step of a small server: one new token for each of 48 requests.
        dict(_plan_case(48, 6000, 48, 64, "decode"), name="plan_decode_48"),
        # A large step: a thousand requests, prompts among the decoding ones.
        dict(_plan_case(1000, 9000, 20011, 16, "mixed"), name="plan_mixed_1000"),
        # A decode step's queries and keys, views of one QKV buffer.
        dict(_rope_case(24, 32, 8, 128, 128), name="rope_decode_24"),
        # A prompt's, an odd number of tokens.
        dict(_rope_case(8191, 32, 8, 128, 128), name="rope_prompt_8191"),
        # An image transformer's joint sequence: as many key heads, adjacent pairs rotated, fp16.
        dict(_rope_case(4173, 20, 20, 64, 64, True, "fp16"), name="rope_image_4173"),
        # One token a request into pages that are part full.
        dict(_append_case(96, 4000, 96, "decode", 8, 128, 64, "int8"), name="append_decode_96"),
        # Three prompts into fresh pages, and the tail of one begun earlier.
        dict(_append_case(3, 700, 6001, "prompt", 8, 128, 128, "fp8", "fp16"), name="append_prompt_6001"),
        # One user's chat, one token: hardly any work, all latency.
        dict(_attend_case(1, 700, 1, "decode", 32, 8, 128, 64, "int8"), name="attend_chat_700"),
        # A decode step over requests of very different lengths.
        dict(_attend_case(40, 12001, 40, "decode", 32, 8, 128, 64, "int8"), name="attend_decode_40"),
        # One token over a long document, eight queries a key head.
        dict(_attend_case(1, 131071, 1, "decode", 64, 8, 128, 128, "fp8"), name="attend_long_131071"),
        # Two whole prompts.
        dict(_attend_case(2, 0, 14003, "prompt", 32, 8, 128, 64, "int8"), name="attend_prompt_14003"),
        # Chunks of prompts beside decoding requests, over a sliding window in small pages.
        dict(_attend_case(12, 9001, 2311, "mixed", 16, 4, 64, 16, "fp8", 4096, "fp16"), name="attend_mixed_2311"),
    ]  # fmt: skip


def _log(rng, low: float, high: float) -> int:
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


HEADS = ((32, 8, 128), (16, 16, 64), (28, 4, 128), (64, 8, 128), (16, 2, 256), (12, 12, 128), (8, 1, 64), (20, 4, 64))


def draw(rng) -> dict:
    op = rng.choice(("plan", "rope", "append", "append", "attend", "attend", "attend", "attend"))
    page = rng.choice((16, 32, 64, 64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    codes = rng.choice(("int8", "fp8"))
    if op == "plan":
        mode = rng.choice(("decode", "mixed", "prompt"))
        requests = _log(rng, 1, 1000)
        tokens = requests if mode == "decode" else requests + _log(rng, 1, 19000)
        return _plan_case(requests, _log(rng, 1, 9000), tokens, page, mode)
    heads, kv_heads, width = rng.choice(HEADS)
    if op == "rope":
        tokens = _log(rng, 1, 8191 * 40 * 128 // ((heads + kv_heads) * width))
        return _rope_case(tokens, heads, kv_heads, width, rng.choice((width, width, width // 2)), rng.random() < 0.3, dtype)
    mode = rng.choice(("decode", "decode", "drafts", "mixed", "prompt"))
    if op == "append":
        requests = _log(rng, 1, 96)
        tokens = {"decode": requests, "drafts": 5 * requests}.get(mode) or requests + _log(rng, 1, 6000)
        tokens = max(requests, min(tokens, 6001 * 1024 // (kv_heads * width)))
        return _append_case(requests, _log(rng, 1, 4000), tokens, mode, kv_heads, width, page, codes, dtype)
    if mode == "prompt":
        requests, longest = rng.randint(1, 4), rng.choice((0, 0, _log(rng, 1, 2000)))
        tokens = _log(rng, 16 * requests, 8192)
    else:
        requests = _log(rng, 1, 64)
        longest = _log(rng, 1, MOST_TOKENS / requests)
        tokens = {"decode": requests, "drafts": rng.randint(2, 8) * requests}.get(mode) or requests + _log(rng, 16, 2000)
    window = rng.choice((0, 0, 0, _log(rng, 16, 8192)))
    case = _attend_case(requests, longest, tokens, mode, heads, kv_heads, width, page, codes, window, dtype)
    while True:
        held, new = _lengths(case)
        pairs = requests * max(new) * (max(held) + max(new)) * heads
        if (pairs <= MOST_PAIRS and work(case)["flops"] <= MOST_WORK) or case["tokens"] <= requests:
            return case
        case["tokens"] = max(requests, case["tokens"] * 2 // 3)


def _lengths(case) -> tuple[list[int], list[int]]:
    """Tokens that each request holds before the step and brings to it: spread over the range by
    the golden ratio, the first the longest; a request in seven holds nothing. `decode` brings one
    each, `drafts` equally many, `mixed` one each and the rest to every fourth request, `prompt`
    all of them split unevenly."""
    requests, longest, tokens = case["requests"], case["longest"], case["tokens"]
    golden = (math.sqrt(5) - 1) / 2
    spread = [(1 - i * golden) % 1 if i else 1.0 for i in range(requests)]
    held = [0 if i % 7 == 6 else round(longest * s) for i, s in enumerate(spread)]
    if case["mode"] in ("decode", "drafts"):
        return held, [tokens // requests] * requests
    new = [1] * requests if tokens >= requests else [int(i < tokens) for i in range(requests)]
    rest = tokens - sum(new)
    takers = list(range(0, requests, 4 if case["mode"] == "mixed" else 1))
    share = [0.5 + spread[(i + 1) % requests] for i in takers]
    for i, s in zip(takers, share):
        new[i] += int(rest * s / sum(share))
    new[takers[-1]] += tokens - sum(new)
    return held, new


# ------------------------------------------------------------------------------ inputs


def _rows(gen, tokens, heads, width, dtype):
    """[tokens, heads, width] with a sixteenth of each head's channels four times louder."""
    x = torch.randn(tokens, heads, width, generator=gen, device="cuda")
    x *= 1 + 3 * (torch.rand(heads, width, generator=gen, device="cuda") < 1 / 16)
    return x.to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(case, gen, held, new):
    """The block table and free list of a server that holds `held` tokens a request: its table is as
    wide as the longest request may grow; its pages are numbered in a random order."""
    page, requests = case["page"], case["requests"]
    have = [-(-h // page) for h in held]
    width = max(-(-(h + n) // page) for h, n in zip(held, new)) + 3
    wanted = sum(-(-(h + n) // page) - a for h, n, a in zip(held, new, have))
    count = sum(have) + wanted + 5
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")
    own_pages = at[None, :] < torch.tensor(have, device="cuda")[:, None]
    table[own_pages] = order[: sum(have)]
    free = torch.zeros(count, dtype=torch.int32, device="cuda")
    free[: wanted + 5] = order[sum(have) :]
    return table, free, _ints([wanted + 5]), count


def _quantized(x, codes):
    """Codes and scales of pages [pages, heads, ...]: the scale is the largest magnitude over the
    format's largest code."""
    scale = (x.abs().amax((2, 3)) / MOST_CODE[codes]).clamp(min=SCALE_FLOOR)
    q = x / scale[..., None, None]
    return (q.round() if codes == "int8" else q).to(CODES[codes]), scale


def prepare(case: dict, seed: int):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = SimpleNamespace(**case)
    if s.op == "rope":
        s.dtype = DTYPES[s.dtype]
        buffer = _rows(gen, s.tokens, s.heads + 2 * s.kv_heads, s.width, s.dtype)
        s.q, s.k = buffer[:, : s.heads], buffer[:, s.heads : s.heads + s.kv_heads]
        s.q_gain, s.k_gain = (1 + 0.1 * torch.randn(2, s.width, generator=gen, device="cuda")).to(s.dtype).unbind(0)
        angle = torch.arange(2 * s.tokens + 500, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(s.rotated // 2, device="cuda") / (s.rotated // 2)
        )
        s.cos, s.sin = angle.cos(), angle.sin()
        s.positions = torch.randint(0, 2 * s.tokens + 500, (s.tokens,), generator=gen, device="cuda", dtype=torch.int32)
        return s
    held, new = _lengths(case)
    s.table, s.free, s.spare, count = _pages(case, gen, held, new)
    s.held, s.new, s.most = _ints(held), _ints(new), max(new)
    if s.op == "plan":
        return s
    s.dtype = DTYPES[s.dtype]
    s.planned = _plain_plan(s)
    shape = (count, s.kv_heads, s.page, s.width)
    filled = torch.arange(count * s.page, device="cuda") < 0  # slots that hold a token
    if s.op == "attend":
        held = [h + n for h, n in zip(held, new)]
        s.longest = max(held)
        s.table = s.planned["table"]
    at = torch.arange(s.table.shape[1] * s.page, device="cuda")
    slot = s.table.long()[:, at // s.page] * s.page + at % s.page
    filled[slot[at[None, :] < torch.tensor(held, device="cuda")[:, None]]] = True
    filled = filled.view(count, 1, s.page, 1)
    k = torch.randn(shape, generator=gen, device="cuda")
    k *= (1 + 3 * (torch.rand(1, s.kv_heads, 1, s.width, generator=gen, device="cuda") < 1 / 16)) * filled
    s.k, s.k_scale = _quantized(k, s.codes)
    v = torch.randn(shape, generator=gen, device="cuda") * filled
    s.v, s.v_scale = _quantized(v, s.codes)
    s.v = s.v.view(torch.int8).transpose(2, 3).contiguous().view(CODES[s.codes])
    if s.op == "append":
        buffer = _rows(gen, s.tokens, 2 * s.kv_heads, s.width, s.dtype)
        s.new_k, s.new_v = buffer[:, : s.kv_heads], buffer[:, s.kv_heads :]
        # The pages of the step's runs, which are read back: whoever plans a step has them.
        s.pages = s.planned["runs"][:, 2].contiguous()
    else:
        s.q = _rows(gen, s.tokens, s.heads, s.width, s.dtype)
    return s


# ------------------------------------------------------------------------------ one pass


def run(s):
    if not own:
        return {"plan": _plain_plan, "rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[s.op](s)
    from cozyq import heads, kv_cache

    if s.op == "rope":
        return heads.norm_rope(torch, s.q, s.k, s.q_gain, s.k_gain, s.cos, s.sin, s.positions, eps=EPS,
                               interleaved=s.interleaved)  # fmt: skip
    if s.op == "plan":
        p = kv_cache.plan(torch, s.table, s.free, s.spare, s.held, s.new, tokens=s.tokens, page=s.page, most=s.most)
        return {"table": p.table, "starts": p.starts, "lengths": p.lengths, "positions": p.positions,
                "requests": p.requests, "slots": p.slots, "runs": p.runs, "spare": p.spare}  # fmt: skip
    cache = kv_cache.PagedCache(s.k, s.v, s.k_scale, s.v_scale)
    p = kv_cache.Plan(page=s.page, most=s.most, **s.planned)
    if s.op == "append":
        cache.append(torch, s.new_k, s.new_v, p)
        return cache.read(torch, s.pages, s.dtype)
    return cache.attend(torch, s.q, p, window=s.window)


def _plain_plan(s):
    """The step's plan in torch's integer operations. Requests' new tokens stand one after another in
    the step's rows. A page whose first slot a new token takes comes off the end of the free list."""
    page, tokens = s.page, s.tokens
    requests, width = s.table.shape
    held, new = s.held.long().clamp(min=0), s.new.long().clamp(min=0)
    zero = torch.zeros(1, dtype=torch.long, device=held.device)
    starts = torch.cat((zero, new.cumsum(0))).clamp(max=tokens)
    lengths = held + starts.diff()
    have = ((held + page - 1) // page).clamp(max=width)
    need = (lengths + page - 1) // page
    taken = torch.cat((zero, (need.clamp(max=width) - have).cumsum(0)))
    row = torch.arange(tokens, device=held.device)
    request = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    valid, at = request < requests, request.clamp(max=requests - 1)
    position = held[at] + row - starts[at]
    index = position // page
    place = taken[at] + index - have[at]
    spare = s.spare.long()
    popped = s.free.long()[(spare - 1 - place).clamp(0, s.free.numel() - 1)]
    popped = torch.where(place < spare, popped, -1)
    kept = s.table.long()[at, index.clamp(max=width - 1)]
    number = torch.where(index >= width, -1, torch.where(index >= have[at], popped, kept))
    slot = torch.where(number >= 0, number * page + position % page, -1)
    first = valid & ((row == starts[at]) | (position % page == 0))
    most = min(tokens, tokens // page + 2 * requests)
    run = torch.where(first, first.cumsum(0) - 1, most)
    count = torch.minimum(starts[at + 1] - row, page - position % page)
    runs = torch.zeros(most + 1, 4, dtype=torch.long, device=held.device)
    runs[:, 2] = -1
    runs[run] = torch.stack((row, count, number, position % page), 1)
    fresh = first & (index >= have[at]) & (index < width)
    table = torch.cat((s.table.long().flatten(), zero))
    table[torch.where(fresh, at * width + index, requests * width)] = number
    got = torch.minimum(taken[-1:], spare)
    left = torch.cat((spare - got, (need - have).sum().reshape(1) - got))
    out = {"table": table[:-1].view(requests, width), "starts": starts, "lengths": lengths,
           "positions": torch.where(valid, position, 0), "requests": torch.where(valid, request, -1),
           "slots": torch.where(valid, slot, -1), "runs": runs[:-1], "spare": left}  # fmt: skip
    return {name: t.to(torch.int32) for name, t in out.items()}


def _plain_rope(s):
    cos, sin = s.cos[s.positions.long()][:, None], s.sin[s.positions.long()][:, None]
    half = s.rotated // 2

    def one(x, gain):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.float()
        turn, rest = x[..., : s.rotated], x[..., s.rotated :]
        if s.interleaved:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = turn[..., :half], turn[..., half:]
            turn = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turn, rest), -1).to(s.dtype)

    return one(s.q, s.q_gain), one(s.k, s.k_gain)


def _rounded(x, codes):
    """What the format's codes hold of `x`, as float32."""
    most = MOST_CODE[codes]
    return x.round().clamp(-most, most) if codes == "int8" else x.clamp(-most, most).to(CODES[codes]).float()


def _plain_append(s):
    """The pages of the step's runs with their new tokens. A run that begins its page clears it; any
    other scales what the page holds again where a new token is larger than its scale reaches."""
    row, count, number, offset = s.planned["runs"].long().unbind(1)
    at = torch.arange(s.page, device=row.device)
    mine = (at >= offset[:, None]) & (at < (offset + count)[:, None])
    token = (row[:, None] + at - offset[:, None]).clamp(0, s.tokens - 1)
    pages = number.clamp(min=0)

    def one(x, codes, scale):
        new = torch.where(mine[:, None, :, None], x.float()[token].transpose(1, 2), 0.0)
        old_scale = torch.where((offset > 0)[:, None], scale[pages], 0.0)
        reach = (new.abs().amax((2, 3)) / MOST_CODE[s.codes]).clamp(min=SCALE_FLOOR)
        scale = torch.maximum(old_scale, reach)[..., None, None]
        old = torch.where((offset > 0)[:, None, None, None], codes[pages].float(), 0.0)
        old = _rounded(old * (old_scale[..., None, None] / scale), s.codes)
        got = torch.where(mine[:, None, :, None], _rounded(new / scale, s.codes), old) * scale
        return torch.where((number >= 0)[:, None, None, None], got, 0.0).to(s.dtype)

    return (one(s.new_k, s.k, s.k_scale),
            one(s.new_v, s.v.view(torch.int8).transpose(2, 3).view(CODES[s.codes]), s.v_scale))  # fmt: skip


def _plain_attend(s):
    """Every request's rows against its pages in one padded rectangle, masked, in float32."""
    requests, group = s.requests, s.heads // s.kv_heads
    count = -(-s.longest // s.page)
    pages = s.table[:, :count].long().clamp(min=0)
    k = (s.k[pages].float() * s.k_scale[pages][..., None, None]).permute(0, 2, 1, 3, 4)
    k = k.reshape(requests * s.kv_heads, count * s.page, s.width)
    v = (s.v[pages].float() * s.v_scale[pages][..., None, None]).permute(0, 2, 1, 4, 3)
    v = v.reshape(requests * s.kv_heads, count * s.page, s.width)
    starts, lengths = s.planned["starts"].long(), s.planned["lengths"].long()
    new = starts.diff()
    i = torch.arange(s.most, device=new.device)
    token = (starts[:-1, None] + i).clamp(max=s.tokens - 1)
    q = s.q.float()[token].view(requests, s.most, s.kv_heads, group, s.width).transpose(1, 2)
    score = torch.bmm(q.reshape(requests * s.kv_heads, s.most * group, s.width), k.transpose(1, 2).contiguous())
    score = score.view(requests, s.kv_heads, s.most, group, -1) * s.width**-0.5
    position = (lengths - new)[:, None] + i
    at = torch.arange(count * s.page, device=new.device)
    seen = (at <= position[..., None]) & (at < lengths[:, None, None])
    if s.window:
        seen &= at > position[..., None] - s.window
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.bmm(score.view(requests * s.kv_heads, s.most * group, -1), v)
    out = out.view(requests, s.kv_heads, s.most, group, s.width) / torch.where(total > 0, total, 1.0)
    out = out.transpose(1, 2).reshape(requests * s.most, s.heads, s.width)
    request = s.planned["requests"].long().clamp(min=0)
    return out[request * s.most + torch.arange(s.tokens, device=new.device) - starts[request]].to(s.dtype)


# ------------------------------------------------------------------------------ work


def work(case: dict) -> dict:
    """Each input once, each output once."""
    c = SimpleNamespace(**case)
    if c.op == "rope":
        values = c.tokens * (c.heads + c.kv_heads) * c.width
        return {"bytes": 4 * values + c.tokens * 4 * (c.rotated + 1), "flops": 7 * values}
    held, new = _lengths(case)
    runs = sum(-(-(h + n) // c.page) - h // c.page for h, n in zip(held, new) if n)
    if c.op == "plan":
        return {"bytes": 4 * (5 * c.requests + 3 * c.tokens + 6 * runs), "flops": 0}
    if c.op == "append":
        values = 2 * c.tokens * c.kv_heads * c.width
        back = 2 * runs * c.kv_heads * c.page * c.width
        return {"bytes": 3 * values + 3 * back, "flops": 3 * values + back}
    seen = pairs = 0
    for h, n in zip(held, new):
        first = max(0, h + 1 - c.window) if c.window else 0
        seen += h + n - first if n else 0
        pairs += sum(min(h + i + 1, c.window or h + i + 1) for i in range(n))
    return {"bytes": 2 * seen * c.kv_heads * c.width + 4 * c.tokens * c.heads * c.width,
            "flops": 4 * pairs * c.heads * c.width}  # fmt: skip


# ------------------------------------------------------------------------------ 64 bits


def exact(case: dict, seed: int):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if s.op == "rope":
        return _exact_rope(s)
    return _exact_append(s) if s.op == "append" else _exact_attend(s)


def _exact_rope(s):
    """As complex numbers: each pair, after its head's norm, times the table's e^(i angle)."""
    turn = torch.complex(s.cos.double(), s.sin.double())[s.positions.long()][:, None]
    out = []
    for x, gain in ((s.q, s.q_gain), (s.k, s.k_gain)):
        x = x.double()
        x = gain.double() * x / (x.square().sum(-1, keepdim=True) / s.width + EPS).sqrt()
        head = x[..., : s.rotated]
        pairs = head.unflatten(-1, (-1, 2)) if s.interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        x[..., : s.rotated] = (turned if s.interleaved else turned.transpose(-1, -2)).flatten(-2)
        out.append(x)
    return out


def _exact_append(s):
    out = []
    most = MOST_CODE[s.codes]
    runs = s.planned["runs"].cpu().tolist()
    for x, codes, scales in ((s.new_k, s.k.float(), s.k_scale), (s.new_v, s.v.float().transpose(2, 3), s.v_scale)):
        got = torch.zeros(len(runs), s.kv_heads, s.page, s.width, dtype=torch.float64, device="cuda")
        for i, (row, count, number, offset) in enumerate(runs):
            if number < 0 or not count:
                continue
            new = x[row : row + count].double().transpose(0, 1)
            scale = (new.abs().amax((1, 2)) / most).clamp(min=SCALE_FLOOR)
            if offset:
                before = scales[number].double()
                scale = torch.maximum(scale, before)
                ratio = (before / scale)[:, None, None]
                got[i] = codes[number].double() * ratio
            got[i, :, offset : offset + count] = new / scale[:, None, None]
            if s.codes == "int8":
                kept = got[i].round().clamp(-most, most)
            else:  # three bits of significand, steps of 2^-9 at the least
                step = torch.exp2(torch.floor(torch.log2(got[i].abs().clamp(min=2.0**-6))) - 3)
                kept = ((got[i] / step).round() * step).clamp(-most, most)
            got[i] = kept * scale[:, None, None]
        out.append(got)
    return out


def _exact_attend(s):
    out = torch.zeros(s.tokens, s.heads, s.width, dtype=torch.float64, device="cuda")
    starts, lengths = s.planned["starts"].tolist(), s.planned["lengths"].tolist()
    group = s.heads // s.kv_heads
    for r in range(s.requests):
        first, last, length = starts[r], starts[r + 1], lengths[r]
        if first == last:
            continue
        pages = s.table[r, : -(-length // s.page)].long()
        at = torch.arange(length, device="cuda")
        position = length - (last - first) + torch.arange(last - first, device="cuda")
        hidden = at > position[:, None]
        if s.window:
            hidden |= at <= position[:, None] - s.window
        for h in range(s.kv_heads):
            k = s.k[pages, h].double() * s.k_scale[pages, h].double()[:, None, None]
            v = s.v[pages, h].double() * s.v_scale[pages, h].double()[:, None, None]
            k, v = k.flatten(0, 1)[:length], v.transpose(1, 2).flatten(0, 1)[:length]
            for g in range(h * group, (h + 1) * group):
                score = s.q[first:last, g].double() @ k.T / math.sqrt(s.width)
                out[first:last, g] = score.masked_fill_(hidden, -math.inf).softmax(-1) @ v
    return out
