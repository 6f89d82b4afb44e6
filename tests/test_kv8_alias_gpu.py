"""Calls whose arrays are the cache's own."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv8(cuda_lib):
    from pvlc_b200 import kv8
    return kv8


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("what", ["advance", "ahead", "both"])
@pytest.mark.parametrize("slots", [5, 1500])
def test_grow_by_the_rows_that_it_changes(kv8, what, slots):
    """advance and ahead are read before tokens is written: every sequence grows by what it held, at
    the edge of its table (42 + 42 + 42 rows of 3 pages and 31)."""
    rng = np.random.default_rng(slots)
    lengths = [int(x) for x in rng.integers(0, 43, slots)]
    lengths[-1] = 42
    c = R.filled_cache(kv8, "int8", lengths, 1, seed=30, spare=3 * slots, room=2)
    assert c.max_pages == 3
    ref, ws = R.Ref(c, "int8"), kv8.Workspace(c, slots)
    advance, ahead = what != "ahead", what != "advance"
    kv8.grow(c, ints(range(slots)), ws, advance=c.tokens if advance else 0,
             ahead=c.tokens if ahead else 0)
    free = iter(np.flatnonzero(ref.refs == 0))
    for s, n in enumerate(lengths):
        ref.tokens[s] = n * (1 + advance)
        for j in range(ref.tokens[s] // 32, (ref.tokens[s] + n * ahead) // 32):
            if ref.table[s, j] < 0:
                ref.table[s, j] = next(free)
                ref.refs[ref.table[s, j]] = 1
    assert ws.errors() == 0
    ref.same(c, pages=False)


def test_grow_slots_that_are_the_row_counts(kv8):
    """slot, too: sequences that hold as many rows as their slot's number."""
    c = R.filled_cache(kv8, "e4m3", [0, 1, 2, 3], 1, seed=31, spare=9)
    ref, ws = R.Ref(c, "e4m3"), kv8.Workspace(c, 4)
    kv8.grow(c, c.tokens, ws, advance=c.tokens, ahead=40)
    assert ws.errors() == 0
    ref.grow([0, 1, 2, 3], [0, 1, 2, 3], [40] * 4)
    ref.same(c)
