"""The examples' command lines, as far as they go without a GPU."""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest


@pytest.fixture
def decode(monkeypatch):
    path = Path(__file__).resolve().parents[1] / "examples" / "decode.py"
    spec = importlib.util.spec_from_file_location("decode_example_cli", path)
    module = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, "decode_example_cli", module)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("name", ["layers", "requests", "prompt", "steps"])
@pytest.mark.parametrize("value", ["0", "-3"])
def test_decode_refuses_counts_below_one(decode, monkeypatch, capsys, name, value):
    def built(*args, **kwargs):
        raise AssertionError("a server was built")

    monkeypatch.setattr(decode, "Server", built)
    monkeypatch.setattr(sys, "argv", ["decode.py", f"--{name}", value])
    with pytest.raises(SystemExit) as left:
        decode.main()
    assert left.value.code == 2 and f"--{name}" in capsys.readouterr().err
