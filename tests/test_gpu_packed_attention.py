"""attention.packed_attention against a float64 softmax over the dequantized cache, element by element.

The bound of an output, as a share of sum_j p_j |v_j|. A rounding to bf16 (8 significant bits) is off by up to half a step,
2^-8 of the value, and there are two on the way: each p v_scale, and the output. (A row that sees one key shows both: its
output is round(round(v_scale) code).) Together (1 + 2^-8)^2 - 1 = 2^-7 + 2^-16. The rest is small: the query's second e4m3
part loses at most 2^-18 of its column's largest element, which moves a score of 128 products by less than 2^-18 * 5 * 128
/ sqrt(128) = 2^-12 and so p by 2^-12 of itself, twice (p and the sum); the exponential is off by 2^-22 and the rounding
of its argument, |s| 2^-24 with |s| < 2^7. In all below 2^-7 + 2^-16 + 2^-11 + 2^-16 < 2^-7 (1 + 2^-3.8)."""
import random

import numpy as np
import pytest
import torch

from nanochat_amd.attention import decode_attention, packed_attention, packed_workspace_bytes, prefill_attention
from nanochat_amd.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu
BOUND = 2.0 ** -7 * (1 + 2.0 ** -3.8)
PAGE = 16


def filled_cache(num_pages, hkv, device, seed):
    """Every slot of the pool holds a token (what a recycled page holds past its sequence's end)."""
    gen = torch.Generator().manual_seed(seed)
    cache = PagedKVCache(num_pages, hkv, device)
    k, v = (torch.randn(1, num_pages * PAGE, hkv, 128, generator=gen).to(torch.bfloat16).to(device) for _ in range(2))
    table = torch.arange(num_pages, dtype=torch.int32, device=device)[None].contiguous()
    cache.append(k, v, torch.zeros(1, dtype=torch.int32, device=device), table)
    return cache


def rows_of(pages, kind):
    """Page bytes [.., 2048] -> e4m3 values [.., 16, 128] in float64."""
    d, slot = torch.arange(128), torch.arange(16)[:, None]
    at = ((d % 32 // 16) * 1024 + (d // 32 * 16 + slot) * 16 + d % 16 if kind == "k" else
          d // 64 * 1024 + (slot // 4 * 16 + d % 16) * 16 + d // 16 % 4 * 4 + slot % 4)
    return pages.cpu()[..., at].view(torch.float8_e4m3fn).double()


def reference(q, cache, table, cu, lens, window, scale=128 ** -0.5):
    """float64 outputs and sum_j p_j |v_j| of every covered row; uncovered rows NaN."""
    k, v = rows_of(cache.k_pages, "k"), rows_of(cache.v_pages, "v")
    s = cache.kv_scale.double().cpu()
    k, v = k * s[:, :, 0, :, None], v * s[:, :, 1, :, None]           # pages, Hkv, 16, 128
    hq, hkv = q.size(1), cache.num_kv_heads
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    size = out.clone()
    qd = q.double().cpu()
    for b in range(len(lens)):
        lo, hi, length = cu[b], cu[b + 1], lens[b]
        if hi == lo:
            continue
        pages = table[b, :-(-length // PAGE)].long().cpu()
        kb, vb = (t[pages].transpose(1, 2).flatten(0, 1)[:length] for t in (k, v))    # keys, Hkv, 128
        p = torch.arange(length - (hi - lo), length)[:, None]
        key = torch.arange(length)
        hidden = key > p
        if window >= 0:
            hidden = hidden | (key < p - window)
        for h in range(hq):
            z = (qd[lo:hi, h] @ kb[:, h * hkv // hq].T * scale).masked_fill(hidden, -torch.inf)
            w = torch.softmax(z, -1)
            out[lo:hi, h] = w @ vb[:, h * hkv // hq]
            size[lo:hi, h] = w @ vb[:, h * hkv // hq].abs()
    return out, size


def setup(device, new, ctx, hq, hkv, seed=0, spare=0, pad_rows=0):
    lens = [n + c for n, c in zip(new, ctx)]
    counts = [-(-length // PAGE) for length in lens]
    rng = random.Random(seed)
    perm = list(range(sum(counts) + spare))
    rng.shuffle(perm)
    table = torch.full((len(new), max(max(counts), 1) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
        at += n
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(cu[-1] + pad_rows, hq, 128, generator=gen).to(torch.bfloat16).to(device)
    cache = filled_cache(max(len(perm), 1), hkv, device, seed + 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return q, cache, table.to(device), ints(cu), ints(lens), cu, lens


def check(got, want, size, cu):
    got = got.double().cpu()
    rows = slice(0, cu[-1])
    worst = float(((got - want).abs() - BOUND * size)[rows].max())
    assert worst <= 1e-6, worst


@pytest.mark.parametrize("hq,hkv", [(4, 4), (16, 4), (6, 6), (12, 4), (10, 2), (16, 1), (13, 13)])
@pytest.mark.parametrize("window", [-1, 0, 5, 100])
def test_mixed_rows(device, hq, hkv, window):
    """Every kind at once: one token and none, a few, chunks that end inside pages and tiles, with and without context."""
    new = [1, 0, 7, 150, 1, 33, 2, 64, 16]
    ctx = [0, 40, 300, 17, 1000, 0, 15, 129, 31]
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, hq, hkv, seed=hq + window)
    got = packed_attention(q, cache, table, cu, lens, max(lens_l), window)
    check(got, *reference(q, cache, table, cu_l, lens_l, window), cu_l)


@pytest.mark.parametrize("n", [1, 2, 3, 8, 9, 15, 16, 17, 31, 32, 33, 65, 127, 128, 129, 257])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 31, 2047, 2049, 4500])
def test_one_sequence(device, n, ctx):
    """Lengths around every border of tiles, pages and chunks; the longer ones in several chunks."""
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [n], [ctx], 8, 2, seed=n + ctx)
    got = packed_attention(q, cache, table, cu, lens, lens_l[0] + 3)
    check(got, *reference(q, cache, table, cu_l, lens_l, -1), cu_l)


@pytest.mark.parametrize("window", [-1, 2500, 333])
def test_long_context_in_many_chunks(device, window):
    new, ctx = [1, 5, 40, 300], [20011, 9000, 17000, 12345]
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 4, 2, seed=3)
    got = packed_attention(q, cache, table, cu, lens, 40000 if table.size(1) >= 2500 else max(lens_l), window)
    check(got, *reference(q, cache, table, cu_l, lens_l, window), cu_l)


def test_many_items_take_tickets(device):
    """More items than workgroups, narrow and wide, twice on one workspace."""
    rng = random.Random(4)
    new = [rng.choice([1, 1, 2, 40, 90]) for _ in range(300)]
    ctx = [rng.randint(0, 60) for _ in new]
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 4, 4, seed=4)
    ws = torch.zeros(packed_workspace_bytes(q.size(0), 300, 4, 4, max(lens_l)), dtype=torch.uint8, device=device)
    got = packed_attention(q, cache, table, cu, lens, max(lens_l), workspace=ws)
    check(got, *reference(q, cache, table, cu_l, lens_l, -1), cu_l)
    again = packed_attention(q, cache, table, cu, lens, max(lens_l), workspace=ws)
    assert torch.equal(got, again)


def test_most_sequences(device):
    new = [b % 3 for b in range(1024)]
    ctx = [b % 37 for b in range(1024)]
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 2, 2, seed=5)
    got = packed_attention(q, cache, table, cu, lens, max(max(lens_l), 1))
    check(got, *reference(q, cache, table, cu_l, lens_l, -1), cu_l)


def test_bits_do_not_depend_on_the_batch(device):
    new, ctx = [1, 9, 200, 3, 70], [5000, 4100, 3000, 0, 6000]
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 8, 2, seed=6)
    whole = packed_attention(q, cache, table, cu, lens, max(lens_l))
    for b in range(5):
        rows = slice(cu_l[b], cu_l[b + 1])
        alone = packed_attention(q[rows].contiguous(), cache, table[b:b + 1].contiguous(),
                                 torch.tensor([0, new[b]], dtype=torch.int32, device=device), lens[b:b + 1].contiguous(),
                                 max(lens_l))
        assert torch.equal(alone, whole[rows]), b


def test_agrees_with_the_padded_forms(device):
    """One token a sequence: decode_attention; equal chunks: prefill_attention. Both within their own bounds of float64."""
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [1] * 6, [0, 3, 100, 1500, 33, 64], 16, 4, seed=7)
    a = packed_attention(q, cache, table, cu, lens, max(lens_l)).float()
    b = decode_attention(q, cache, table, lens, max(lens_l)).float()
    want, size = reference(q, cache, table, cu_l, lens_l, -1)
    assert float(((a - b).abs().cpu() - 2 * BOUND * size).max()) <= 1e-6
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [40] * 3, [7, 160, 0], 8, 2, seed=8)
    a = packed_attention(q, cache, table, cu, lens, max(lens_l)).float()
    b = prefill_attention(q.view(3, 40, 8, 128), cache, table, lens - 40).float().flatten(0, 1)
    want, size = reference(q, cache, table, cu_l, lens_l, -1)
    assert float(((a - b).abs().cpu() - 2 * BOUND * size).max()) <= 1e-6


def test_rows_behind_the_last_sequence_stay(device):
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [3, 0, 50], [9, 5, 5], 4, 2, seed=9, pad_rows=11)
    out = torch.full_like(q, 5.0)
    assert packed_attention(q, cache, table, cu, lens, max(lens_l), out=out) is out
    check(out, *reference(q, cache, table, cu_l, lens_l, -1), cu_l)
    assert bool((out[53:] == 5.0).all())


@pytest.mark.parametrize("n", [1, 20, 150])
def test_stale_slots_and_pages(device, n):
    """Infinities and NaN in the scales of slots past the sequence's end, in pages of nobody, and in later rows' own keys
    reach no row that does not see them."""
    hq, hkv, ctx = 4, 2, 21
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [n], [ctx], hq, hkv, seed=10, spare=3)
    want, size = reference(q, cache, table, cu_l, lens_l, -1)
    length = n + ctx
    last = int(table[0, (length - 1) // PAGE])
    if length % PAGE:
        cache.kv_scale[last, :, :, length % PAGE:] = float("inf")
        cache.kv_scale[last, :, 1, length % PAGE] = float("nan")
        cache.k_pages[last].view(hkv, 2, 4, 16, 16)[:, :, :, length % PAGE:] = 0x7F     # NaN codes
        cache.v_pages[last].view(hkv, 2, 4, 16, 4, 4)[:, :, length % PAGE // 4, :, :, length % PAGE % 4:] = 0x7F
    used = set(table[0, :-(-length // PAGE)].tolist())
    for page in set(range(cache.num_pages)) - used:
        cache.kv_scale[page] = float("nan")
    got = packed_attention(q, cache, table, cu, lens, length)
    check(got, want, size, cu_l)
    if n > 2:      # a NaN key and an infinite value at the middle row's position: the rows before it do not see them
        mid = ctx + n // 2
        page, slot = int(table[0, mid // PAGE]), mid % PAGE
        cache.kv_scale[page, :, 0, slot], cache.kv_scale[page, :, 1, slot] = float("nan"), float("inf")
        got = packed_attention(q, cache, table, cu, lens, length)
        check(got[:n // 2], want[:n // 2], size[:n // 2], [0, n // 2])
        assert bool(torch.isnan(got[n // 2:]).all())


def test_what_does_not_fit_becomes_nan(device):
    """Lengths past max_seq_len or below the new tokens, and entries outside the pool: NaN for those, the rest right."""
    new, ctx = [4, 1, 60, 1, 90, 2], [50, 900, 100, 30, 10, 3]
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 4, 2, seed=11)
    want, size = reference(q, cache, table, cu_l, lens_l, -1)
    lens[3], lens[5] = 0, 1
    table[0, 1], table[4, 0] = cache.num_pages, -1
    out = torch.zeros_like(q)
    packed_attention(q, cache, table, cu, lens, 500, out=out)
    for b, bad in enumerate([True, True, False, True, True, True]):
        rows = slice(cu_l[b], cu_l[b + 1])
        if bad:
            assert bool(torch.isnan(out[rows]).all()), b
        else:
            check(out[rows], want[rows], size[rows], [0, new[b]])


def test_row_offsets_out_of_order_stay_in_bounds(device):
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [40] * 8, [3000] * 8, 4, 2, seed=12, pad_rows=5)
    before = q.clone()
    for offsets in ([0, 400, 0, 400, 0, 400, 0, 400, 0], [-5, 2 ** 31 - 1, 7, 9, 3, -2 ** 31, 0, 320, 325],
                    [320, 280, 240, 200, 160, 120, 80, 40, 0]):
        guard = torch.full((q.size(0) + 2, 4, 128), 3.0, dtype=torch.bfloat16, device=device)
        packed_attention(q, cache, table, torch.tensor(offsets, dtype=torch.int32, device=device), lens, max(lens_l),
                         out=guard[1:-1])
        assert bool((guard[0] == 3.0).all()) and bool((guard[-1] == 3.0).all())
    assert torch.equal(q, before)
    got = packed_attention(q, cache, table, cu, lens, max(lens_l))          # the workspace's counts are as they were
    check(got, *reference(q, cache, table, cu_l, lens_l, -1), cu_l)


def test_captured(device):
    """One graph for steps of other lengths, eager calls between the replays; its workspace is its own."""
    new, ctx = [1, 30, 0, 140, 2], [4000, 2500, 3, 5000, 0]
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 8, 2, seed=13)
    out = torch.empty_like(q)
    packed_attention(q, cache, table, cu, lens, 5160, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed_attention(q, cache, table, cu, lens, 5160, out=out)
    for other in ([1, 30, 0, 140, 2], [140, 1, 30, 2, 0], [0, 0, 173, 0, 0], [1, 1, 1, 1, 1]):
        held = [min(n + 37 * b, lens_l[b]) if n else lens_l[b] for b, n in enumerate(other)]
        held = [max(h, n) if max(h, n) <= lens_l[b] else lens_l[b] for b, (h, n) in enumerate(zip(held, other))]
        other = [min(n, h) for n, h in zip(other, held)]
        offsets = np.concatenate([[0], np.cumsum(other)]).tolist()
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        lens.copy_(torch.tensor(held, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        eager = packed_attention(q, cache, table, cu, lens, 5160)
        torch.cuda.synchronize()
        assert torch.equal(out[:offsets[-1]], eager[:offsets[-1]])
        check(out, *reference(q, cache, table, offsets, held, -1), offsets)


def test_refusals(device):
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [2, 1], [3, 4], 4, 2)
    run = lambda **k: packed_attention(**{**dict(q=q, cache=cache, block_table=table, cu_seqlens=cu, seq_lens=lens,  # noqa: E731
                                                 max_seq_len=16), **k})
    run()
    for bad in (dict(q=q[:, :3].contiguous()), dict(q=q[:, :, :64].contiguous()), dict(q=q[0]), dict(q=q.cpu()), dict(q=q[:, ::2]),
                dict(cu_seqlens=cu[:2]), dict(seq_lens=lens[:1]), dict(seq_lens=lens.cpu()), dict(max_seq_len=0),
                dict(max_seq_len=10 ** 6), dict(out=q[:2].clone()), dict(block_table=table[:1]),
                dict(workspace=torch.zeros(64, dtype=torch.uint8, device=device))):
        with pytest.raises(ValueError):
            run(**bad)
    for bad in (dict(q=q.float()), dict(cu_seqlens=cu.long()), dict(block_table=table.long())):
        with pytest.raises(TypeError):
            run(**bad)
    assert run(q=q[:0]).shape == (0, 4, 128)
