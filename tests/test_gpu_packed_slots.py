"""attention.packed_attention over more sequences than one launch takes (1,024): as many as a paging.BlockTables has slots."""
import pytest
import torch

from nanochat_amd.attention import packed_attention, packed_workspace_bytes
from nanochat_amd.kv_cache import PagedKVCache
from nanochat_amd.paging import BlockTables

from .test_gpu_packed_attention import check, reference, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,window", [(1025, -1), (2048, 9), (2500, -1), (4096, -1)])
def test_many_sequences(device, batch, window):
    new = [0 if b % 3 == 1 else 1 + 39 * (b % 256 == 5) for b in range(batch)]
    ctx = [b % 37 for b in range(batch)]
    ctx[1024] = 2300                                     # a cut sequence in the second launch
    new[1024] = 2
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 2, 1, seed=batch, pad_rows=3)
    want, size = reference(q, cache, table, cu_l, lens_l, window)
    out = torch.full_like(q, 5.0)
    assert packed_attention(q, cache, table, cu, lens, max(lens_l), window, out=out) is out
    check(out, want, size, cu_l)
    assert bool((out[cu_l[-1]:] == 5.0).all())
    need = packed_workspace_bytes(q.size(0), batch, 2, 1, max(lens_l), window)
    ws = torch.zeros(need, dtype=torch.uint8, device=device)
    for _ in range(2):
        assert torch.equal(packed_attention(q, cache, table, cu, lens, max(lens_l), window, workspace=ws)[:cu_l[-1]],
                           out[:cu_l[-1]])


def test_as_many_slots_as_block_tables_have(device):
    """extend's maps for 4,096 slots as they are, eager and captured."""
    slots = 4096
    tables = BlockTables(slots, 4, 2 * slots, device)
    cache = PagedKVCache(2 * slots, 1, device)
    cache.kv_scale.fill_(1.0)
    cache.v_pages.fill_(0x38)                            # every value 1
    new = torch.ones(slots, dtype=torch.int32, device=device)
    q = torch.zeros(slots, 1, 128, dtype=torch.bfloat16, device=device)
    maps = tables.extend(new, slots)
    out = packed_attention(q, cache, tables.table, maps.cu_seqlens, tables.lengths, 64)
    assert bool((out == 1.0).all())
    out.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        maps = tables.extend(new, slots, maps)
        packed_attention(q, cache, tables.table, maps.cu_seqlens, tables.lengths, 64, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert bool((out == 1.0).all())


def test_refusals_name_the_limit(device):
    q, cache, table, cu, lens, _, _ = setup(device, [2, 1], [3, 4], 17, 1)
    with pytest.raises(ValueError, match="at most 16 query heads a KV head"):
        packed_attention(q, cache, table, cu, lens, 16)


@pytest.mark.parametrize("shift", [1, 2, 3, 4])
def test_tensors_at_any_offset(device, shift):
    """Contiguous views that start at no multiple of 16 bytes: rows, row offsets, lengths and the table."""
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [1, 30, 4, 90], [2400, 100, 0, 700], 6, 2, seed=shift)
    moved = lambda t, n: torch.cat([t.new_zeros(n), t.flatten()])[n:].view(t.shape)  # noqa: E731
    out = moved(torch.zeros_like(q), 5 - shift)
    got = packed_attention(moved(q, shift), cache, moved(table, shift), moved(cu, shift), moved(lens, 1), max(lens_l), out=out)
    assert torch.equal(got, packed_attention(q, cache, table, cu, lens, max(lens_l)))
