"""How attention to an encoder's states cuts the steps of few rows into runs, on the CPU by the kernels' own sums and
rules (`cozyq_host_cross_runs`): every run that a join reads has its places in the workspace, whatever `starts` holds."""

from __future__ import annotations

import random

import numpy as np
import pytest

from cozyq import _lib

MANY = 1 << 30


def runs(tokens, q_heads, states, kv_heads, width, most, starts, lengths):
    """(total steps, a run's, places, first run, last run), or None where nothing is cut."""
    starts, lengths = (np.ascontiguousarray(x, dtype=np.int32) for x in (starts, lengths))
    out = np.zeros(5, dtype=np.int32)
    assert len(starts) == len(lengths) + 1
    cut = _lib.load().cozyq_host_cross_runs(tokens, q_heads, len(lengths), states, kv_heads, width, most,
                                            starts.ctypes.data, lengths.ctypes.data, out.ctypes.data)  # fmt: skip
    assert cut in (0, 1)
    return tuple(map(int, out)) if cut else None


def held(found):
    total, run, places, first, last = found
    assert total >= 0 and run >= 8 and 0 <= first <= last < places, found


def test_starts_in_any_order_stay_within_the_workspace():
    """A request in two claims all of the call's rows: 64 tiles' steps beyond 2^30 twice over, of which a sum of more than
    kMany, as each 64 requests come to, has no place in 32 bits."""
    tokens, requests = 80000, 128
    starts = [tokens * (i % 2) for i in range(requests + 1)]
    for most in (1, 4, 8):
        found = runs(tokens, 32, 64000, 8, 128, most, starts, [64000] * requests)
        held(found)
        assert found[0] == MANY and found[1] > MANY // found[2]
    for requests in (64, 65, 256, 3000):
        starts = [tokens * (i % 2) for i in range(requests + 1)]
        held(runs(tokens, 8, 64000, 8, 64, 1, starts, [64000] * requests))
        held(runs(tokens, 8, 64000, 8, 64, 1, [2**31 - 1, -5] * (requests // 2) + [0] * (1 + requests % 2), [2**31 - 1] * requests))


@pytest.mark.parametrize("seed", range(6))
def test_ascending_and_shuffled_starts(seed):
    """The runs hold every step of requests in order, and of others no run past the last is read."""
    rng = random.Random(seed)
    for _ in range(40):
        requests = rng.choice((1, 2, 7, 63, 64, 65, 200, 700))
        rows = [rng.choice((0, 1, 1, 3, 8)) for _ in range(requests)]
        tokens, states = sum(rows), rng.choice((800, 1600, 6400, 30000, 100000))
        kv_heads, group = rng.choice((1, 3, 8, 20)), rng.choice((1, 4))
        width = rng.choice((40, 64, 128, 256))
        starts = [sum(rows[:i]) for i in range(requests + 1)]
        lengths = [rng.choice((0, 1, states, rng.randint(0, states))) for _ in rows]
        most = max(1, max(rows))
        found = runs(tokens, kv_heads * group, states, kv_heads, width, most, starts, lengths)
        if not found:
            continue
        held(found)
        tile = 32 if most * group > 16 else 16
        steps = sum(-(-n * group // tile) * max(1, -(-length // 32)) for n, length in zip(rows, lengths))
        assert found[0] == steps
        rng.shuffle(starts)
        held(runs(tokens, kv_heads * group, states, kv_heads, width, most, starts, lengths))


def test_calls_of_more_threads_than_a_launch_has_are_refused():
    """2^32 threads: 256 a tile of 16 rows and key head, and 512 one of 256."""
    size = _lib.load().cozyq_cross_attend_workspace_bytes
    assert size(65535, 4096, 65535, 10, 4096, 64, 1) == -1
    assert size(65535, 256, 65535, 10, 256, 64, 1) == -1 and size(65535, 128, 65535, 10, 128, 64, 1) == 0
    assert size(1 << 23, 256, 1, 10, 256, 8, 0) == -1 and size(1 << 22, 256, 1, 10, 256, 8, 0) == 0
    one, at = np.zeros(32, dtype=np.float32), np.zeros(1, dtype=np.int32)
    p = one.ctypes.data + -one.ctypes.data % 16
    call = _lib.load().cozyq_cross_attend
    assert call(0, p, 0, 65535, 4096, 64, 64, p, p, 65535, 10, 4096, 64, 64, 64, 64, 64, 64, 64, at.ctypes.data, None, None, 0, 1,
                1.0, p, None, None) == 1  # fmt: skip
