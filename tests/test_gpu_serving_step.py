"""The operators of one continuous-batching step run together, as a server's loop would: BlockTables.extend, the packed
append, packed attention, a product with a head, sample_tokens, BlockTables.trim. Each step's tables, cache bytes, attention
outputs and tokens are checked against their oracles; then the same step captured into a graph, two at once on two streams,
and pools and logits past 2^31 bytes."""
import numpy as np
import pytest
import torch

import oracle.paging
from nanochat_amd.attention import packed_attention, qk_norm_rope_append_packed
from nanochat_amd.kv_cache import PagedKVCache
from nanochat_amd.paging import BlockTables
from nanochat_amd.rotary import rotary_tables
from nanochat_amd.sampling import sample_tokens
from oracle.token_choice import choose
from tests.test_gpu_packed_append import check as check_cache, expect, filled, oracle_of
from tests.test_gpu_packed_attention import check as check_attention, reference
from tests.test_gpu_sampling import NEAR

pytestmark = pytest.mark.gpu
VOCAB = 9001


class Server:
    """One layer and a head with random weights; `rows` packed rows a step."""

    def __init__(self, device, slots, max_pages, num_pages, rows, hq, hkv, seed=0):
        gen = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.hq, self.hkv, self.rows, self.slots = hq, hkv, rows, slots
        self.tables = BlockTables(slots, max_pages, num_pages, device)
        self.tables.free_pages.copy_(torch.randperm(num_pages, generator=gen).to(torch.int32))
        self.cache = filled(device, num_pages, hkv, seed)
        self.gains = [(1 + 0.1 * rand(128)).to(device) for _ in range(2)]
        self.cos, self.sin = (t.to(device) for t in rotary_tables(max_pages * 16))
        self.head = (rand(hq * 128, VOCAB) / 8).to(torch.bfloat16).to(device)
        self.max_len = max_pages * 16

    def step(self, qkv, new, uniform, temperature, top_k, top_p, window=-1):
        maps = self.tables.extend(new, self.rows)
        q = qk_norm_rope_append_packed(qkv, self.hq, self.cache, maps.positions, maps.slot_map, *self.gains, self.cos,
                                       self.sin)
        out = packed_attention(q, self.cache, self.tables.table, maps.cu_seqlens, self.tables.lengths, self.max_len, window)
        last = (maps.cu_seqlens[1:] - 1).clamp(min=0).long()          # a slot's last row; its token is used if it had any
        logits = out.flatten(1)[last] @ self.head
        return maps, q, out, logits, sample_tokens(logits, uniform, temperature, top_k, top_p)


def inputs(server, device, seed):
    gen = torch.Generator().manual_seed(seed)
    n = server.slots
    qkv = torch.randn(server.rows, (server.hq + 2 * server.hkv) * 128, generator=gen).to(torch.bfloat16).to(device)
    u = torch.rand(n, generator=gen).to(device)
    t = torch.where(torch.rand(n, generator=gen) < 0.3, 0.0, 0.9).to(device)
    k = torch.randint(0, 60, (n,), generator=gen, dtype=torch.int32).to(device)
    return qkv, u, t, k, torch.full((n,), 0.9, device=device)


@pytest.mark.parametrize("hq,hkv,window", [(4, 4, -1), (8, 2, 40), (5, 1, -1)])
def test_steps_match_the_oracles(device, hq, hkv, window):
    """Prompts, then decoding with drafts of which some are taken back, slots that finish and start again, a pool that runs
    out of pages in between."""
    slots, max_pages, num_pages, rows = 6, 20, 44, 150
    s = Server(device, slots, max_pages, num_pages, rows, hq, hkv)
    paging = oracle.paging.BlockTables(slots, max_pages, num_pages)
    paging.free = s.tables.free_pages.tolist()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    plan = [([40, 0, 17, 3, 1, 0], None), ([4, 90, 1, 1, 1, 20], [-1, -1, 18, 4, -1, -1]), ([1, 4, 1, 130, 1, 1], [43, 91, 0, -1, -1, 21]),
            ([1, 3, 100, 1, 2, 1], [-1, 93, -1, -1, -1, -1]), ([1, 1, 1, 140, 1, 1], [-1, -1, -1, 0, -1, -1]), ([2, 1, 1, 55, 1, 1], None)]
    for i, (new, keep) in enumerate(plan):
        qkv, *settings = inputs(s, device, i)
        o = oracle_of(s.cache)
        marker = torch.zeros(rows, hq, 128, device=device)
        maps, q, out, logits, tokens = s.step(qkv, ints(new), *settings, window)
        cu, positions, slot_map, granted = paging.extend(new, rows)
        assert maps.cu_seqlens.tolist() == cu and maps.granted.tolist() == granted
        assert maps.positions.tolist() == positions and maps.slot_map.tolist() == slot_map
        assert s.tables.lengths.tolist() == paging.lengths and s.tables.table.tolist() == paging.table
        live = cu[-1]
        want = expect(o, qkv, hq, hkv, *s.gains, s.cos, s.sin, maps.positions, maps.slot_map, marker)
        check_cache(s.cache, o, q[:live], want[:live])
        table = s.tables.table.clone()
        ref, size = reference(q, s.cache, table, cu, paging.lengths, window)
        check_attention(out[:live], ref[:live], size[:live], cu)
        z = logits.float().cpu().numpy()
        for b in range(slots):
            if granted[b]:
                u, t, k, p = (float(x[b]) for x in settings)
                token, margin = choose(z[b], u, t, int(k), p)
                assert margin < NEAR or tokens[b].item() == token
        if keep is not None:
            s.tables.trim(ints(keep))
            paging.trim(keep)
            assert s.tables.lengths.tolist() == paging.lengths
            assert s.tables.free_pages[:s.tables.free_count.item()].tolist() == paging.free


def test_captured_step(device):
    """One graph of the whole step and its trim, replayed with other inputs; an eager twin runs between the replays."""
    make = lambda: Server(device, 5, 30, 150, 64, 8, 2, seed=3)  # noqa: E731
    a, b = make(), make()
    new, keep = (torch.zeros(5, dtype=torch.int32, device=device) for _ in range(2))
    static = inputs(a, device, 0)

    def step(server, args):
        maps, q, out, logits, tokens = server.step(args[0], new, *args[1:])
        server.tables.trim(keep)
        return maps, out, tokens

    keep.fill_(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, static)              # no new tokens: only loads what the step needs
        step(b, static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a, static)
    lengths = [0] * 5
    for i in range(5):
        counts = [[30, 5, 0, 1, 9], [1, 1, 40, 1, 4], [1, 4, 1, 2, 1], [1, 1, 1, 50, 1], [3, 0, 1, 1, 0]][i]
        lengths = [x + c for x, c in zip(lengths, counts)]
        kept = [x - 1 if c > 3 else -1 for x, c in zip(lengths, counts)]
        lengths = [x - 1 if c > 3 else x for x, c in zip(lengths, counts)]
        new.copy_(torch.tensor(counts, dtype=torch.int32))
        keep.copy_(torch.tensor(kept, dtype=torch.int32))
        fresh = inputs(a, device, 20 + i)
        for x, y in zip(static, fresh):
            x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        want = step(b, fresh)
        torch.cuda.synchronize()
        live = sum(counts)
        for x, y in zip(got[0], want[0]):
            assert torch.equal(x, y)
        assert torch.equal(got[1][:live], want[1][:live])
        had = torch.tensor(counts, device=device) > 0
        assert torch.equal(got[2][had], want[2][had])
        assert a.tables.lengths.tolist() == b.tables.lengths.tolist() == lengths
        assert torch.equal(a.cache.k_pages, b.cache.k_pages) and torch.equal(a.cache.kv_scale, b.cache.kv_scale)


def test_two_streams_and_two_graphs(device):
    """Attention in partials and rows in slices, whose workgroups count on one another through a workspace: eager calls on
    two streams at once, then two graphs replayed at once, give what each gives alone."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    sides = []
    for seed in (5, 6):
        s = Server(device, 8, 300, 2400, 200, 8, 2, seed)
        gen = torch.Generator().manual_seed(seed)
        ctx = torch.tensor([4700, 3000, 2500, 1, 600, 4000, 100, 2200], dtype=torch.int32, device=device)
        s.tables.extend(ctx, 20000)
        new = torch.tensor([1, 4, 90, 1, 3, 1, 60, 2], dtype=torch.int32, device=device)
        maps = s.tables.extend(new, 200)
        q = torch.randn(200, 8, 128, generator=gen).to(torch.bfloat16).to(device)
        logits = torch.randn(40, 40000, generator=gen).to(device)
        u, t, p = torch.rand(40, generator=gen).to(device), torch.ones(40, device=device), torch.full((40,), 0.9, device=device)
        k = torch.randint(0, 200, (40,), generator=gen, dtype=torch.int32).to(device)

        def call(s=s, q=q, maps=maps, logits=logits, u=u, t=t, k=k, p=p):
            out = torch.zeros_like(q)
            packed_attention(q, s.cache, s.tables.table, maps.cu_seqlens, s.tables.lengths, s.max_len, out=out)
            return out, sample_tokens(logits, u, t, k, p)
        sides.append(call)
    s = None
    want = [call() for call in sides]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(sides[i]())
    torch.cuda.synchronize()
    same = lambda x, y: torch.equal(x[0].view(torch.int16), y[0].view(torch.int16)) and torch.equal(x[1], y[1])  # noqa: E731
    for i in range(2):
        assert all(same(r, want[i]) for r in results[i])
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(sides[i]())
    for _ in range(10):
        for out in outs:
            out[0].zero_(), out[1].zero_()
        torch.cuda.synchronize()
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert same(outs[i], want[i])
        assert same(sides[0](), want[0])


def test_pool_past_2_31_bytes(device):
    """The pages of a pool whose byte offsets need more than 32 bits, against the same pages in a small pool."""
    hq, hkv, big, small = 4, 4, 540_000, 60          # 540,000 x 4 x 2 KiB = 4.4e9 bytes of K
    rows = 300
    gen = torch.Generator().manual_seed(9)
    qkv = torch.randn(rows, (hq + 2 * hkv) * 128, generator=gen).to(torch.bfloat16).to(device)
    cos, sin = (t.to(device) for t in rotary_tables(400))
    gain = torch.ones(128, device=device)
    out = []
    for pages, first in ((small, 0), (big, big - small)):
        cache = PagedKVCache(pages, hkv, device)
        tables = BlockTables(4, 30, small, device)
        maps = tables.extend(torch.tensor([200, 1, 40, 59], dtype=torch.int32, device=device), rows)
        slot_map = torch.where(maps.slot_map < 0, -1, maps.slot_map + first * 16).to(torch.int32)
        table = torch.where(tables.table < 0, -1, tables.table + first).to(torch.int32)
        q = qk_norm_rope_append_packed(qkv, hq, cache, maps.positions, slot_map, gain, gain, cos, sin)
        out.append((q, packed_attention(q, cache, table, maps.cu_seqlens, tables.lengths, 480),
                    cache.k_pages[first:first + small].clone(), cache.v_pages[first:first + small].clone(),
                    cache.kv_scale[first:first + small].clone()))
        del cache
    held = torch.unique(tables.table[tables.table >= 0]).long()
    for i, (x, y) in enumerate(zip(*out)):
        if i >= 2:
            x, y = x[held], y[held]
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), i


def test_logits_past_2_31_elements(device):
    rows, vocab, stride = 4, 9000, 2 ** 30
    buffer = torch.empty((rows - 1) * stride + vocab, dtype=torch.bfloat16, device=device)
    logits = buffer.as_strided((rows, vocab), (stride, 1))
    gen = torch.Generator().manual_seed(10)
    values = torch.randn(rows, vocab, generator=gen).to(torch.bfloat16).to(device)
    logits.copy_(values)
    u, t = torch.rand(rows, generator=gen).to(device), torch.ones(rows, device=device)
    p = torch.full((rows,), 0.8, device=device)
    assert torch.equal(sample_tokens(logits, u, t, top_p=p), sample_tokens(values, u, t, top_p=p))
