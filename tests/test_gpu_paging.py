"""paging.BlockTables against the integer oracle: every output, the tables, lengths and free list after every call."""
import random

import pytest
import torch

from nanochat_amd.paging import BlockTables
from oracle import paging as oracle

pytestmark = pytest.mark.gpu


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def same_state(t, o):
    assert t.table.tolist() == o.table
    assert t.lengths.tolist() == o.lengths
    assert int(t.free_count) == len(o.free) and t.free_pages[:len(o.free)].tolist() == o.free


@pytest.mark.parametrize("slots,max_pages,num_pages,rows,biggest", [
    (1, 1, 1, 1, 3), (1, 40, 40, 700, 600), (7, 5, 20, 64, 40), (64, 8, 300, 64, 2), (256, 9, 900, 3000, 60),
    (257, 3, 700, 513, 17), (1000, 4, 2500, 9001, 33), (4096, 2, 5000, 4096, 2)])
def test_steps_match_the_oracle(device, slots, max_pages, num_pages, rows, biggest):
    rng = random.Random(slots)
    t, o = BlockTables(slots, max_pages, num_pages, device), oracle.BlockTables(slots, max_pages, num_pages)
    for _ in range(12):
        asked = [rng.choice([0, 1, -1, rng.randint(0, biggest)]) for _ in range(slots)]
        got, want = t.extend(ints(asked, device), rows), o.extend(asked, rows)
        for name, g, w in zip(got._fields, got, want):
            assert g.tolist() == w, name
        same_state(t, o)
        keep = [rng.choice([-1, -1, n + 1, n, 0, n // 2, n - 1]) for n in o.lengths]
        t.trim(ints(keep, device))
        o.trim(keep)
        same_state(t, o)


def test_trim_undoes_extend(device):
    t = BlockTables(50, 20, 600, device)
    t.extend(ints([(7 * b) % 90 for b in range(50)], device), 5000)
    before = [x.clone() for x in (t.table, t.lengths, t.free_pages, t.free_count)]
    lengths = t.lengths.clone()
    t.extend(ints([(11 * b) % 60 for b in range(50)], device), 5000)
    t.trim(lengths)
    for x, y in zip(before, (t.table, t.lengths, t.free_pages, t.free_count)):
        assert torch.equal(x, y)


def test_numbers_at_the_ends_of_int32(device):
    """Requests whose sums pass 32 bits are refused, the others served."""
    t, o = BlockTables(4096, 2, 64, device), oracle.BlockTables(4096, 2, 64)
    big = [2 ** 31 - 1, -2 ** 31, 31, 2 ** 31 - 1] * 1024
    got, want = t.extend(ints(big, device), 40), o.extend(big, 40)
    for g, w in zip(got, want):
        assert g.tolist() == w
    same_state(t, o)
    t = BlockTables(1, 2 ** 27 - 1, 4, device)          # a row of 2^31 - 16 positions
    assert t.extend(ints([2 ** 31 - 1], device), 8).granted.tolist() == [0]
    assert t.extend(ints([5], device), 8).granted.tolist() == [5]


def test_captured_steps(device):
    """Extend and trim in one graph, replayed with other requests, eager work between the replays."""
    slots, rows = 33, 200
    t, o = BlockTables(slots, 6, 120, device), oracle.BlockTables(slots, 6, 120)
    asked, keep = torch.zeros(slots, dtype=torch.int32, device=device), torch.full((slots,), -1, dtype=torch.int32, device=device)
    maps = t.extend(asked, rows)                        # a step that asks nothing, before the capture
    t.trim(keep)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.extend(asked, rows, maps)
        t.trim(keep)
    rng = random.Random(1)
    for _ in range(6):
        a = [rng.randint(0, 12) for _ in range(slots)]
        k = [rng.choice([-1, 0, 5]) for _ in range(slots)]
        asked.copy_(ints(a, device))
        keep.copy_(ints(k, device))
        torch.cuda.synchronize()
        graph.replay()
        want = o.extend(a, rows)
        o.trim(k)
        for g, w in zip(maps, want):
            assert g.tolist() == w
        same_state(t, o)
        t.extend(torch.zeros_like(asked), rows)
        torch.cuda.synchronize()


def test_refusals(device):
    t = BlockTables(4, 4, 8, device)
    with pytest.raises(ValueError, match="new_tokens"):
        t.extend(torch.zeros(5, dtype=torch.int32, device=device), 4)
    with pytest.raises(TypeError, match="new_tokens"):
        t.extend(torch.zeros(4, dtype=torch.int64, device=device), 4)
    with pytest.raises(ValueError, match="rows"):
        t.extend(torch.zeros(4, dtype=torch.int32, device=device), 0)
    with pytest.raises(ValueError, match="keep"):
        t.trim(torch.zeros(4, dtype=torch.int32))
    maps = t.extend(torch.zeros(4, dtype=torch.int32, device=device), 4)
    with pytest.raises(ValueError, match="positions"):
        t.extend(torch.zeros(4, dtype=torch.int32, device=device), 5, maps)
    with pytest.raises(ValueError, match="share memory"):   # read by every workgroup while one writes what was granted
        t.extend(maps.granted, 4, maps)
    t.extend(maps.granted, 4)
    t.extend(t.lengths, 4, maps)                            # lengths are written after everyone has read them
