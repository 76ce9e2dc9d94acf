"""The page bookkeeping oracle: every page is free or held once, refusals, and the rollback."""
import random

import pytest

from oracle.paging import PAGE, BlockTables, pages_of


def consistent(t, num_pages):
    held = []
    for row, length in zip(t.table, t.lengths):
        assert all(p >= 0 for p in row[:pages_of(length)]) and all(p == -1 for p in row[pages_of(length):])
        held += row[:pages_of(length)]
    assert sorted(held + t.free) == list(range(num_pages))


@pytest.mark.parametrize("seed", range(5))
def test_pages_are_never_lost_or_shared(seed):
    rng = random.Random(seed)
    t = BlockTables(9, 6, 30)
    for _ in range(60):
        asked = [rng.choice([0, 1, 1, 5, 17, 40, -2]) for _ in range(9)]
        before = list(t.lengths)
        cu, positions, slot_map, granted = t.extend(asked, 70)
        consistent(t, 30)
        assert [b - a for a, b in zip(cu, cu[1:])] == granted and cu[-1] <= 70
        assert all(g in (0, max(n, 0)) for g, n in zip(granted, asked))
        live = [s for s in slot_map if s >= 0]
        assert len(live) == len(set(live)) == cu[-1] and len(positions) == 70
        for b in range(9):
            assert positions[cu[b]:cu[b + 1]] == list(range(before[b], before[b] + granted[b]))
        t.trim([rng.choice([-1, 0, n, max(n - 3, 0)]) for n in t.lengths])
        consistent(t, 30)


def test_refusals():
    t = BlockTables(4, 2, 3)
    assert t.extend([16, 17, 1, 0], 100)[3] == [16, 17, 0, 0]        # the third page is the last one
    assert t.extend([0, 15, 1, 5], 100)[3] == [0, 15, 0, 0]          # a slot that needs no page is served
    assert t.extend([17, 1, 0, 0], 100)[3] == [0, 0, 0, 0]           # past the table's row; no page left
    t.trim([0, -1, -1, -1])
    assert t.extend([3, 0, 2, 0], 4)[3] == [3, 0, 0, 0]              # the page goes to slot 0, none is left for slot 2
    t = BlockTables(3, 2, 6)
    assert t.extend([3, 2, 1], 4)[3] == [3, 0, 0]                    # rows: from the first slot that does not fit on


def test_trim_undoes_extend():
    t = BlockTables(3, 4, 12)
    t.extend([5, 33, 16], 100)
    table, lengths, free = [list(r) for r in t.table], list(t.lengths), list(t.free)
    t.extend([20, 1, 30], 100)
    t.trim(lengths)
    assert (t.table, t.lengths, t.free) == (table, lengths, free)
    assert PAGE == 16
