"""`examples/describe.py`: the residual norm, positions on three axes and attention to an encoder's states as one model
uses them, beside the paged cache and the int8 linears."""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest
import torch

from oracle import cache as law
from oracle import layer as laws
from test_gpu_cross import check as check_cross
from test_gpu_kv_cache import DEV, check_rope
from test_gpu_norms import check as check_norm


@pytest.fixture
def example(monkeypatch):
    path = Path(__file__).resolve().parents[1] / "examples" / "describe.py"
    spec = importlib.util.spec_from_file_location("describe_example", path)
    module = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, "describe_example", module)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("name", ["layers", "requests", "side", "prompt", "states", "steps"])
@pytest.mark.parametrize("value", ["0", "-2"])
def test_counts_below_one_are_refused(example, monkeypatch, capsys, name, value):
    def built(*args, **kwargs):
        raise AssertionError("a server was built")

    monkeypatch.setattr(example, "Describer", built)
    monkeypatch.setattr(sys, "argv", ["describe.py", f"--{name}", value])
    with pytest.raises(SystemExit) as left:
        example.main()
    assert left.value.code == 2 and f"--{name}" in capsys.readouterr().err


SHAPE = dict(layers=2, requests=3, q_heads=8, kv_heads=2, width=64, side=4, states=150, encoder=256, page=16, pages=24, longest=96)  # fmt: skip


@pytest.mark.gpu
def test_each_operator_of_a_prompt_is_near_its_formula(example, monkeypatch):
    """The layers over three prompts, every call of the operators held against 64 bits on its own inputs, by the bars of
    the operators' own tests."""
    server = example.Describer(**SHAPE)
    server.seen[1] = 0  # a request without an image
    calls = {"norm": 0, "rope": 0, "cross": 0}
    add_rms, norm_rope, cross = example.norms.add_rms, example.heads.norm_rope, example.attention.cross

    def checked_norm(t, x, residual, gain):
        operand, total = add_rms(t, x, residual, gain)
        check_norm(operand, total, x, residual, gain, torch.int8)
        calls["norm"] += 1
        return operand, total

    def checked_rope(t, q, k, q_gain, k_gain, cos, sin, positions, *, sections, cycled):
        got = norm_rope(t, q, k, q_gain, k_gain, cos, sin, positions, sections=sections, cycled=cycled)
        own = laws.tables(cos.cpu(), sin.cpu(), positions.cpu(), sections, cycled)
        for x, gain, y in zip((q, k), (q_gain, k_gain), got):
            check_rope(y, *law.norm_rope(x.cpu(), gain.cpu(), *own, None, 1e-6, False), x.dtype)
        calls["rope"] += 1
        return got

    def checked_cross(t, q, k, v, *, starts, lengths, most):
        got = cross(t, q, k, v, starts=starts, lengths=lengths, most=most)
        check_cross(got, q, k, v, starts, lengths)
        calls["cross"] += 1
        return got

    monkeypatch.setattr(example.norms, "add_rms", checked_norm)
    monkeypatch.setattr(example.heads, "norm_rope", checked_rope)
    monkeypatch.setattr(example.attention, "cross", checked_cross)
    x = torch.randn(20 + 37 + 1, 512, generator=torch.Generator(DEV).manual_seed(5), device=DEV).bfloat16()
    y = server.prompt(x, [20, 37, 1])
    assert y.isfinite().all() and calls == {"norm": 4, "rope": 2, "cross": 2}
    axes = server.axes(server.plan(torch.ones(3, dtype=torch.int32, device=DEV), 3, 1)).tolist()
    assert axes == [[8, 25, 0], [8, 25, 0], [8, 25, 1]]  # text, text, the second patch


@pytest.mark.gpu
def test_recorded_steps_are_those_taken_eagerly(example):
    """Steps replayed from a graph against the same steps run eagerly in a second server, over page boundaries and
    other lengths of the states: the same kernels on the same numbers, so the same bits."""
    lengths, steps = [30, 16, 1], 20
    gen = torch.Generator(DEV).manual_seed(72)
    prompt = torch.randn(sum(lengths), 512, generator=gen, device=DEV).bfloat16()
    tokens = torch.randn(steps, 3, 512, generator=gen, device=DEV).bfloat16()
    a, b = example.Describer(**SHAPE), example.Describer(**SHAPE)
    assert torch.equal(a.prompt(prompt, lengths), b.prompt(prompt, lengths))
    x, y, graph = a.recorded_step()
    one = torch.ones(3, dtype=torch.int32, device=DEV)
    b.forward(torch.zeros_like(x), b.plan(one, 3, 1))  # the recorded server has run its step once before it was recorded
    for t in range(steps):
        for server in (a, b):
            server.seen.copy_(torch.tensor([150 - t, 7 * t, 0 if t % 2 else 33]))
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
