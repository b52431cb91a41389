"""A language model that reads images: its layers attend to their own tokens, at positions on three axes, through the
8-bit paged cache, and to an encoder's states; between the linears runs one residual stream, normed into their operands.

    python examples/describe.py [--layers 4 --requests 16 --side 16 --prompt 100 --states 1600 --steps 64]

Each request begins with `side` x `side` image patches, at (0, row, column), and goes on with text, at one position on
all axes. Weights and states are random, projections int8.convrot; the MLP is left out. Every request has the states of
an encoder of its own, the first fewest. One token a request and step is recorded into a HIP graph once and replayed.
"""

from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path
from typing import Any

import torch

sys.path[:0] = [str(Path(__file__).resolve().parents[1] / "cozy-runtime_amd"), str(Path(__file__).resolve().parent)]

from cozyq import attention, encode, heads, int8_linear, norms  # noqa: E402
from decode import Server  # noqa: E402


@dataclass
class Between:
    """What a layer has beside its attention to its own tokens."""

    first: Any  # the norms' gains
    second: Any
    query: tuple
    states: tuple
    out: tuple


class Describer(Server):
    """A `Server` whose layers read `states` encoder states of `encoder` elements a request too."""

    def __init__(self, layers=4, requests=16, q_heads=32, kv_heads=8, width=128, side=16, states=1600, encoder=1024, seed=0, **rest):  # fmt: skip
        super().__init__(layers, requests, q_heads, kv_heads, width, seed=seed, **rest)
        gen = torch.Generator("cuda").manual_seed(seed + 1)

        def weight(n, k):
            made = encode.encode_int8_convrot256(torch, "w", torch.randn(n, k, generator=gen, device="cuda") * k**-0.5)
            return made.payload.view(torch.int8).view(n, k), made.companions[0].raw.view(torch.float32).reshape(-1)

        def gain():
            return (1 + 0.1 * torch.randn(self.hidden, generator=gen, device="cuda")).bfloat16()

        self.side = side
        # Pairs in turns: a quarter of them is of the rows, as many of the columns.
        pairs = width // 2
        self.sections = (pairs - 2 * (pairs // 4), pairs // 4, pairs // 4)
        self.between = [
            Between(gain(), gain(), weight(self.hidden, self.hidden), weight(2 * kv_heads * width, encoder), weight(self.hidden, self.hidden))
            for _ in range(layers)
        ]
        self.states = torch.randn(requests, states, encoder, generator=gen, device="cuda").bfloat16()
        self.seen = torch.linspace(max(1, states // 4), states, requests, device="cuda").int()
        self.look()

    def look(self):
        """The states' keys and values for every layer, once for all of a request's tokens."""
        requests, count, _ = self.states.shape
        self.kept = []
        for layer in self.between:
            both = int8_linear.linear(torch, self.states, *layer.states, None, self.states.dtype)
            both = both.view(requests, count, 2 * self.kv_heads, self.width)
            self.kept.append((both[:, :, : self.kv_heads], both[:, :, self.kv_heads :]))

    def axes(self, plan):
        """The rows' positions on three axes, int32 `[3, T]`."""
        p, patches = plan.positions, self.side**2
        text = p - patches + self.side
        image = torch.stack([torch.zeros_like(p), p // self.side, p % self.side])
        return torch.where(p < patches, image, text)

    def forward(self, x, plan):
        """The layers over the step's rows `x` `[T, hidden]`."""
        tokens, q, kv = x.shape[0], self.q_heads, self.kv_heads
        positions, stream = self.axes(plan), None
        for layer, more, (k, v) in zip(self.layers, self.between, self.kept):
            operand, stream = norms.add_rms(torch, x, stream, more.first)
            qkv = int8_linear.gemm(torch, operand, *layer.qkv, None, x.dtype).view(tokens, q + 2 * kv, self.width)
            queries, keys = heads.norm_rope(torch, qkv[:, :q], qkv[:, q : q + kv], layer.q_gain, layer.k_gain, self.cos, self.sin,
                                            positions, sections=self.sections, cycled=True)  # fmt: skip
            layer.cache.append(torch, keys, qkv[:, q + kv :], plan)
            own = layer.cache.attend(torch, queries, plan)
            x = int8_linear.linear(torch, own.view(tokens, self.hidden), *layer.out, None, x.dtype)
            operand, stream = norms.add_rms(torch, x, stream, more.second)
            queries = int8_linear.gemm(torch, operand, *more.query, None, x.dtype).view(tokens, q, self.width)
            shown = attention.cross(torch, queries, k, v, starts=plan.starts, lengths=self.seen, most=plan.most)
            x = int8_linear.linear(torch, shown.view(tokens, self.hidden), *more.out, None, x.dtype)
        return x + stream


def main() -> None:
    ask = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    counts = (("layers", 4), ("requests", 16), ("side", 16), ("prompt", 100), ("states", 1600), ("steps", 64))
    for name, value in counts:
        ask.add_argument(f"--{name}", type=int, default=value)
    args = ask.parse_args()
    for name, _ in counts:
        if getattr(args, name) < 1:
            ask.error(f"--{name} is at least 1")
    length = args.side**2 + args.prompt
    longest = length + args.steps + 1
    server = Describer(args.layers, args.requests, side=args.side, states=args.states, longest=longest,
                       pages=args.requests * (-(-longest // 64) + 1))  # fmt: skip
    x = torch.randn(args.requests * length, server.hidden, device="cuda").bfloat16()
    server.prompt(x, [length] * args.requests)
    torch.cuda.synchronize()
    print(f"prompts: {len(x)} tokens of {args.requests} requests through {args.layers} layers, each over up to {args.states} states")
    x, y, graph = server.recorded_step()
    for step in range(args.steps + 1):
        if step == 1:  # the first one loads the norm's kernel and the graph
            torch.cuda.synchronize()
            began = time.perf_counter()
        graph.replay()
        x.copy_(torch.nn.functional.rms_norm(y, (server.hidden,)))
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / args.steps
    print(f"{args.steps} steps: {took * 1e6:.1f} us a step, {args.requests / took:.0f} tokens/s")


if __name__ == "__main__":
    main()
