"""attention.qk_norm_rope_append_packed against the oracle (cache bytes, scales and queries bit-exact) and against the
padded append: sequences of mixed lengths, rows in any order, padding rows, strided rows, every other slot of the pool
left as it was."""
import numpy as np
import pytest
import torch

from nanochat_amd.attention import qk_norm_rope_append, qk_norm_rope_append_packed
from nanochat_amd.kv_cache import PagedKVCache
from nanochat_amd.paging import BlockTables
from nanochat_amd.rotary import rotary_tables
from oracle.layout import PAGE, PagedCache
from oracle.quant import quantize_rows
from oracle.rope import qk_norm_rope

pytestmark = pytest.mark.gpu


def make(device, rows, hq, hkv, seed, rope_len=700, pad=0):
    gen = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(rows, (hq + 2 * hkv) * 128 + pad, generator=gen) * 1.5).to(torch.bfloat16)
    gains = [1 + 0.1 * torch.randn(128, generator=gen) for _ in range(2)]
    cos, sin = rotary_tables(rope_len)
    return [t.to(device) for t in (qkv, *gains, cos, sin)]


def filled(device, num_pages, hkv, seed):
    """A pool with something in every byte, so that a store outside the rows' slots shows."""
    gen = torch.Generator().manual_seed(seed)
    cache = PagedKVCache(num_pages, hkv, device)
    for t in (cache.k_pages, cache.v_pages):
        t.copy_(torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8))
    cache.kv_scale.copy_(torch.rand(cache.kv_scale.shape, generator=gen))
    return cache


def oracle_of(cache):
    o = PagedCache(cache.num_pages, cache.num_kv_heads)
    o.k, o.v = cache.k_pages.cpu().numpy().copy(), cache.v_pages.cpu().numpy().copy()
    o.ks, o.vs = cache.k_scale.cpu().numpy().copy(), cache.v_scale.cpu().numpy().copy()
    return o


def check(cache, o, got, want):
    assert np.array_equal(cache.k_pages.cpu().numpy(), o.k) and np.array_equal(cache.v_pages.cpu().numpy(), o.v)
    assert np.array_equal(cache.k_scale.cpu().numpy(), o.ks) and np.array_equal(cache.v_scale.cpu().numpy(), o.vs)
    assert np.array_equal(got.float().cpu().numpy(), want)


def expect(o, qkv, hq, hkv, gq, gk, cos, sin, positions, slot_map, q_before):
    """The oracle's cache and queries; q_before: what skipped rows keep."""
    x = qkv[:, :(hq + 2 * hkv) * 128].float().cpu().numpy().reshape(-1, hq + 2 * hkv, 128)
    pos, slots = positions.cpu().numpy(), slot_map.cpu().numpy()
    live = (pos >= 0) & (pos < cos.size(0)) & (slots >= 0) & (slots < o.k.shape[0] * PAGE)
    want = q_before.float().cpu().numpy().copy()
    if live.any():
        x, pos, slots = x[live], pos[live], slots[live]
        c, s = cos.cpu().numpy()[pos][:, None], sin.cpu().numpy()[pos][:, None]
        want[live] = qk_norm_rope(x[:, :hq], gq.cpu().numpy(), c, s)
        k = qk_norm_rope(x[:, hq:hq + hkv], gk.cpu().numpy(), c, s)
        o.scatter(slots // PAGE, slots % PAGE, *quantize_rows(k), *quantize_rows(x[:, hq + hkv:]))
    return want


@pytest.mark.parametrize("hq,hkv", [(4, 4), (16, 4), (13, 13), (5, 1)])
@pytest.mark.parametrize("new", [[1], [1] * 19, [3, 0, 1, 65, 2, 16, 17], [130, 1, 1, 31]])
def test_matches_the_oracle(device, hq, hkv, new):
    ctx = [(37 * b + 5) % 90 for b in range(len(new))]
    tables = BlockTables(len(new), 20, 20 * len(new), device)
    tables.free_pages.copy_(torch.randperm(20 * len(new), generator=torch.Generator().manual_seed(1)).to(torch.int32))
    tables.extend(torch.tensor(ctx, dtype=torch.int32, device=device), max(sum(ctx), 1))
    rows = sum(new) + 5                                            # five padding rows
    maps = tables.extend(torch.tensor(new, dtype=torch.int32, device=device), rows)
    qkv, gq, gk, cos, sin = make(device, rows, hq, hkv, len(new))
    cache = filled(device, tables.num_pages, hkv, 3)
    o = oracle_of(cache)
    q = torch.full((rows, hq, 128), 7.0, dtype=torch.bfloat16, device=device)
    want = expect(o, qkv, hq, hkv, gq, gk, cos, sin, maps.positions, maps.slot_map, q)
    got = qk_norm_rope_append_packed(qkv, hq, cache, maps.positions, maps.slot_map, gq, gk, cos, sin, q_out=q)
    check(cache, o, got, want)
    assert float(got[-5:].float().min()) == float(got[-5:].float().max()) == 7.0


@pytest.mark.parametrize("order", ["shuffled", "reversed", "shifted"])
def test_rows_in_any_order(device, order):
    """Slots with no runs at all, runs backwards, and runs that start at every slot of a page."""
    hq, hkv, num_pages, rows = 8, 2, 12, 150
    slots = torch.randperm(num_pages * PAGE, generator=torch.Generator().manual_seed(2))[:rows]
    if order == "reversed":
        slots = torch.arange(rows - 1, -1, -1)
    if order == "shifted":
        slots = torch.cat([torch.arange(rows // 2) + 5, torch.arange(rows - rows // 2) + 101])
    positions = (torch.arange(rows) * 3 % 700).to(torch.int32).to(device)
    slot_map = slots.to(torch.int32).to(device)
    qkv, gq, gk, cos, sin = make(device, rows, hq, hkv, 9, pad=24)
    qkv = qkv[:, :(hq + 2 * hkv) * 128]                            # a strided view
    cache = filled(device, num_pages, hkv, 4)
    o = oracle_of(cache)
    q = torch.zeros(rows, hq, 128, dtype=torch.bfloat16, device=device)
    want = expect(o, qkv, hq, hkv, gq, gk, cos, sin, positions, slot_map, q)
    check(cache, o, qk_norm_rope_append_packed(qkv, hq, cache, positions, slot_map, gq, gk, cos, sin), want)


def test_rows_that_are_skipped(device):
    """Slots and positions at and past every end: those rows store nothing, their neighbours in the same quad do."""
    hq, hkv, num_pages = 4, 2, 4
    slots = [0, 1, 2, 3, 4, -1, 6, 7, 8, 9, 64, 11, 12, 13, 14, 2 ** 31 - 1, 16, 17, 18, 19, 63]
    places = [5, 6, 7, 8, 9, 10, 11, 12, -1, 14, 15, 16, 99, 100, 101, 1, -2 ** 31, 99, 98, 2 ** 31 - 1, 0]
    positions = torch.tensor(places, dtype=torch.int32, device=device)
    slot_map = torch.tensor(slots, dtype=torch.int32, device=device)
    qkv, gq, gk, cos, sin = make(device, len(slots), hq, hkv, 10, rope_len=100)
    cache = filled(device, num_pages, hkv, 5)
    o = oracle_of(cache)
    q = torch.full((len(slots), hq, 128), -2.0, dtype=torch.bfloat16, device=device)
    want = expect(o, qkv, hq, hkv, gq, gk, cos, sin, positions, slot_map, q)
    check(cache, o, qk_norm_rope_append_packed(qkv, hq, cache, positions, slot_map, gq, gk, cos, sin, q_out=q), want)


def test_special_rows(device):
    """Zero rows (scale 1), one huge element, the smallest bf16 values."""
    hq, hkv = 2, 1
    qkv, gq, gk, cos, sin = make(device, 6, hq, hkv, 11)
    qkv[0], qkv[1, 300], qkv[2] = 0, 3e38, qkv[2] * 1e-38
    positions = torch.arange(6, dtype=torch.int32, device=device)
    cache = filled(device, 1, hkv, 6)
    o = oracle_of(cache)
    q = torch.zeros(6, hq, 128, dtype=torch.bfloat16, device=device)
    with np.errstate(over="ignore", invalid="ignore"):
        want = expect(o, qkv, hq, hkv, gq, gk, cos, sin, positions, positions, q)
    check(cache, o, qk_norm_rope_append_packed(qkv, hq, cache, positions, positions, gq, gk, cos, sin), want)


def test_same_bits_as_the_padded_append(device):
    hq, hkv, T = 16, 4, 37
    starts = torch.tensor([0, 21, 64], dtype=torch.int32, device=device)
    table = torch.randperm(24, generator=torch.Generator().manual_seed(8)).to(torch.int32).view(3, 8).to(device)
    qkv, gq, gk, cos, sin = make(device, 3 * T, hq, hkv, 12)
    one, two = filled(device, 24, hkv, 7), filled(device, 24, hkv, 7)
    q1 = qk_norm_rope_append(qkv.view(3, T, -1), hq, one, table, starts, gq, gk, cos, sin)
    positions = (starts[:, None] + torch.arange(T, dtype=torch.int32, device=device)).flatten()
    seq = torch.arange(3, device=device).repeat_interleave(T)
    slot_map = table[seq, positions // PAGE] * PAGE + positions % PAGE
    q2 = qk_norm_rope_append_packed(qkv, hq, two, positions, slot_map, gq, gk, cos, sin)
    assert torch.equal(q1.flatten(0, 1), q2)
    for name in ("k_pages", "v_pages", "kv_scale"):
        assert torch.equal(getattr(one, name), getattr(two, name)), name


def test_refusals(device):
    hq, hkv = 4, 2
    qkv, gq, gk, cos, sin = make(device, 3, hq, hkv, 1)
    cache = PagedKVCache(2, hkv, device)
    at = torch.arange(3, dtype=torch.int32, device=device)
    run = lambda **k: qk_norm_rope_append_packed(**{**dict(qkv=qkv, num_q_heads=hq, cache=cache, positions=at, slot_map=at,  # noqa: E731
                                                           q_gain=gq, k_gain=gk, cos=cos, sin=sin), **k})
    run()
    for bad in (dict(num_q_heads=5), dict(qkv=qkv.float()), dict(qkv=qkv.cpu()), dict(positions=at[:2]), dict(slot_map=at.cpu()),
                dict(qkv=qkv[None]), dict(cos=cos[:10]), dict(q_gain=gq[:64]), dict(qkv=qkv[:1].expand(3, -1)),
                dict(q_out=torch.empty(3, 5, 128, dtype=torch.bfloat16, device=device))):
        with pytest.raises(ValueError):
            run(**bad)
    for bad in (dict(positions=at.long()), dict(k_gain=gk.double())):
        with pytest.raises(TypeError):
            run(**bad)
    empty = run(qkv=qkv[:0], positions=at[:0], slot_map=at[:0])
    assert empty.shape == (0, hq, 128)
