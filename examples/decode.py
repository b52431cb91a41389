"""A language model's attention layers on quantized linears and the 8-bit paged cache: prompts in one
step, then one token a request and step, the step recorded into a HIP graph once and replayed.

    python examples/decode.py [--layers 4 --requests 16 --prompt 600 --steps 64 --codes int8|fp8]

Weights are random: int8.convrot projections, made on the GPU from normal matrices. The MLP is left out.
What a server keeps between steps is the block table, the free list, each request's length and the layers'
caches; a step's plan reads and moves all of it on the GPU, so nothing waits for the host.
"""

from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path
from typing import Any

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "cozy-runtime_amd"))

from cozyq import encode, heads, int8_linear, kv_cache  # noqa: E402


@dataclass
class Layer:
    qkv: tuple
    out: tuple
    q_gain: Any
    k_gain: Any
    cache: kv_cache.PagedCache


class Server:
    """`requests` sequences over `layers` attention layers of `q_heads` x `width` queries and `kv_heads` keys."""

    def __init__(self, layers=4, requests=16, q_heads=32, kv_heads=8, width=128, page=64, pages=512, longest=4096,
                 codes=torch.int8, seed=0):  # fmt: skip
        self.q_heads, self.kv_heads, self.width, self.page = q_heads, kv_heads, width, page
        self.hidden = q_heads * width
        gen = torch.Generator("cuda").manual_seed(seed)

        def weight(n, k):
            made = encode.encode_int8_convrot256(torch, "w", torch.randn(n, k, generator=gen, device="cuda") * k**-0.5)
            scale = made.companions[0].raw.view(torch.float32).reshape(-1)
            return made.payload.view(torch.int8).view(n, k), scale

        def gain():
            return (1 + 0.1 * torch.randn(width, generator=gen, device="cuda")).bfloat16()

        self.layers = [
            Layer(weight((q_heads + 2 * kv_heads) * width, self.hidden), weight(self.hidden, self.hidden), gain(), gain(),
                  kv_cache.empty(torch, pages, kv_heads, width, page=page, dtype=codes))  # fmt: skip
            for _ in range(layers)
        ]
        angle = torch.arange(longest, device="cuda")[:, None] * 10000.0 ** (-torch.arange(width // 2, device="cuda") / (width // 2))
        self.cos, self.sin = angle.cos(), angle.sin()
        self.table = torch.full((requests, -(-longest // page)), -1, dtype=torch.int32, device="cuda")
        self.free = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.spare = torch.tensor([pages, 0], dtype=torch.int32, device="cuda")
        self.held = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def plan(self, new, tokens, most, out=None):
        """The step in which request r brings `new[r]` of `tokens` rows."""
        return kv_cache.plan(torch, self.table, self.free, self.spare, self.held, new, tokens=tokens, page=self.page,
                             most=most, out=out)  # fmt: skip

    def commit(self, plan):
        """The step's lengths and free pages become the server's."""
        self.held.copy_(plan.lengths)
        self.spare.copy_(plan.spare)

    def forward(self, x, plan):
        """The layers over the step's rows `x` `[T, hidden]`, each added to its input."""
        tokens, q, kv = x.shape[0], self.q_heads, self.kv_heads
        for layer in self.layers:
            qkv = int8_linear.linear(torch, x, *layer.qkv, None, x.dtype).view(tokens, q + 2 * kv, self.width)
            queries, keys = heads.norm_rope(torch, qkv[:, :q], qkv[:, q : q + kv], layer.q_gain, layer.k_gain, self.cos,
                                            self.sin, plan.positions)  # fmt: skip
            layer.cache.append(torch, keys, qkv[:, q + kv :], plan)
            seen = layer.cache.attend(torch, queries, plan)
            x = x + int8_linear.linear(torch, seen.view(tokens, self.hidden), *layer.out, None, x.dtype)
        return x

    def prompt(self, x, lengths):
        """Prompts of `lengths` tokens, their rows one after another in `x`."""
        new = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        plan = self.plan(new, x.shape[0], max(lengths))
        y = self.forward(x, plan)
        self.commit(plan)
        return y

    def recorded_step(self):
        """(x, y, graph): a replay takes one token a request from x through the layers into y."""
        requests = self.held.shape[0]
        # What the graph reads and writes lives as long as the server does.
        one = self.one = torch.ones(requests, dtype=torch.int32, device="cuda")
        x = torch.zeros(requests, self.hidden, dtype=torch.bfloat16, device="cuda")
        plan = self.step_plan = self.plan(one, requests, 1)  # its tensors, and a first run of every kernel
        self.forward(x, plan)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.plan(one, requests, 1, out=plan)
            y = self.forward(x, plan)
            self.commit(plan)
        return x, y, graph


def main() -> None:
    ask = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 4), ("requests", 16), ("prompt", 600), ("steps", 64)):
        ask.add_argument(f"--{name}", type=int, default=value)
    ask.add_argument("--codes", choices=("int8", "fp8"), default="int8")
    args = ask.parse_args()
    for name in ("layers", "requests", "prompt", "steps"):
        if getattr(args, name) < 1:
            ask.error(f"--{name} is at least 1")
    longest = args.prompt + args.steps + 1
    pages = args.requests * (-(-longest // 64) + 1)
    server = Server(args.layers, args.requests, pages=pages, longest=longest,
                    codes=torch.int8 if args.codes == "int8" else torch.float8_e4m3fn)  # fmt: skip
    lengths = [max(1, args.prompt - 37 * r % args.prompt) for r in range(args.requests)]
    x = torch.randn(sum(lengths), server.hidden, device="cuda").bfloat16()
    y = server.prompt(x, lengths)
    torch.cuda.synchronize()
    print(f"prompts: {sum(lengths)} tokens of {args.requests} requests through {args.layers} layers")
    x, y, graph = server.recorded_step()
    for step in range(args.steps + 1):
        if step == 1:  # the first one loads the norm's kernel and the graph
            torch.cuda.synchronize()
            began = time.perf_counter()
        graph.replay()
        x.copy_(torch.nn.functional.rms_norm(y, (server.hidden,)))
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / args.steps
    print(f"{args.steps} steps: {took * 1e6:.1f} us a step, {args.requests / took:.0f} tokens/s; longest request "
          f"{int(server.held.max())} tokens, {int(server.spare[0])} of {pages} pages free")  # fmt: skip


if __name__ == "__main__":
    main()
