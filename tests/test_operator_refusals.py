"""What the serving operators refuse on the host, before any device call: null pointers and sizes at the C ABI, sizes at
the Python entry points."""
import ctypes

import pytest

from nanochat_amd.paging import BlockTables

DUMMY = ctypes.c_void_p(0x1000)   # never dereferenced: every call below fails its host checks first


def extend_args(**over):
    args = dict(new_tokens=DUMMY, slots=4, lengths=DUMMY, table=DUMMY, max_pages=4, free_pages=DUMMY, free_count=DUMMY,
                num_pages=8, rows=4, cu_seqlens=DUMMY, positions=DUMMY, slot_map=DUMMY, granted=DUMMY, arrived=DUMMY,
                stream=None)
    return list((args | over).values())


def trim_args(**over):
    args = dict(keep=DUMMY, slots=4, lengths=DUMMY, table=DUMMY, max_pages=4, free_pages=DUMMY, free_count=DUMMY,
                num_pages=8, arrived=DUMMY, stream=None)
    return list((args | over).values())


def append_args(**over):
    args = dict(qkv=DUMMY, token_stride=24 * 128, rows=4, Hq=16, Hkv=4, positions=DUMMY, slot_map=DUMMY, q_gain=DUMMY,
                k_gain=DUMMY, cos=DUMMY, sin=DUMMY, rope_len=64, q_out=DUMMY, k_pages=DUMMY, v_pages=DUMMY,
                kv_scale=DUMMY, num_pages=8, stream=None)
    return list((args | over).values())


@pytest.mark.parametrize("name", ["new_tokens", "lengths", "table", "free_pages", "free_count", "cu_seqlens", "positions",
                                  "slot_map", "granted", "arrived"])
def test_extend_rejects_null(lib, name):
    assert lib.nc_pages_extend(*extend_args(**{name: None})) == -1


@pytest.mark.parametrize("over", [dict(slots=0), dict(slots=4097), dict(max_pages=0), dict(num_pages=0), dict(rows=0),
                                  dict(rows=-1), dict(num_pages=2 ** 27), dict(max_pages=2 ** 27)])
def test_extend_rejects_sizes(lib, over):
    assert lib.nc_pages_extend(*extend_args(**over)) == -2


def test_trim_rejects(lib):
    for name in ("keep", "lengths", "table", "free_pages", "free_count", "arrived"):
        assert lib.nc_pages_trim(*trim_args(**{name: None})) == -1, name
    for over in (dict(slots=0), dict(slots=4097), dict(max_pages=0), dict(num_pages=0), dict(num_pages=2 ** 27)):
        assert lib.nc_pages_trim(*trim_args(**over)) == -2, over


def test_append_rows_rejects(lib):
    for name in ("qkv", "positions", "slot_map", "q_gain", "k_gain", "cos", "sin", "q_out", "k_pages", "v_pages", "kv_scale"):
        assert lib.nc_qk_norm_rope_append_rows_fp8(*append_args(**{name: None})) == -1, name
    for over in (dict(rows=-1), dict(rows=2 ** 28), dict(Hq=0), dict(Hkv=0), dict(num_pages=0), dict(num_pages=2 ** 27),
                 dict(rope_len=0), dict(token_stride=24 * 128 - 1)):
        assert lib.nc_qk_norm_rope_append_rows_fp8(*append_args(**over)) == -2, over
    assert lib.nc_qk_norm_rope_append_rows_fp8(*append_args(rows=0)) == 0


def packed_args(**over):
    args = dict(q=DUMMY, k_pages=DUMMY, v_pages=DUMMY, kv_scale=DUMMY, block_table=DUMMY, max_pages=16, num_pages=8,
                cu_seqlens=DUMMY, seq_lens=DUMMY, rows=4, B=2, Hq=16, Hkv=4, max_seq_len=256, window=-1, sm_scale=0.1,
                out=DUMMY, workspace=DUMMY, workspace_bytes=1 << 30, stream=None)
    return list((args | over).values())


def test_packed_attention_rejects(lib):
    for name in ("q", "k_pages", "v_pages", "kv_scale", "block_table", "cu_seqlens", "seq_lens", "out", "workspace"):
        assert lib.nc_packed_attn_fp8(*packed_args(**{name: None})) == -1, name
    for over in (dict(rows=0), dict(rows=2 ** 24 + 1), dict(B=0), dict(B=1025), dict(Hq=6), dict(Hq=68), dict(Hkv=0),
                 dict(max_seq_len=0), dict(max_seq_len=257), dict(max_pages=0), dict(num_pages=0)):
        assert lib.nc_packed_attn_fp8(*packed_args(**over)) == -2, over
    need = lib.nc_packed_workspace_bytes(4096, 64, 16, 4, 8192, -1)
    assert need > 0
    assert lib.nc_packed_attn_fp8(*packed_args(rows=4096, B=64, max_pages=512, max_seq_len=8192,
                                               workspace_bytes=need - 1024)) == -3


def plan(rows, n, length, hq, hkv, window):
    """The cut of a sequence as packed_attn.hip's pk_plan makes it: (units, items, partials a kind)."""
    tpt, page = 16 // (hq // hkv), 16
    first = max(length - n - window, 0) if window >= 0 else 0
    pg0 = first // page & ~1
    pages = (length - 1) // page + 1 - pg0
    if n <= 2 * tpt:
        tiles, cut = 1, 128 if pages <= 128 else 64
    else:
        tiles = (n - 1) // (8 * tpt) + 1
        want = max(256 // (tiles * hkv), 1)
        cut = min(max(((pages - 1) // want + 1 + 31) & ~31, 128), 1024)
    chunks = (pages - 1) // cut + 1
    return (n <= 2 * tpt, tiles * hkv * chunks if chunks > 1 else 0, tiles * hkv if chunks > 1 else 0)


def test_packed_workspace_holds_every_launch(lib):
    """Whatever the lengths, the partials and counts of a launch fit what the host asked for (the kernel refuses the rest)."""
    import random

    rng = random.Random(0)
    for _ in range(3000):
        hq, hkv = rng.choice([(4, 4), (16, 4), (16, 1), (13, 13), (10, 2)])
        batch, most = rng.randint(1, 40), rng.choice([100, 3000, 20000, 70000])
        window = rng.choice([-1, -1, 0, 700, 30000])
        new = [min(rng.choice([0, 1, 3, 33, 200, 3000]), most) for _ in range(batch)]
        rows = max(sum(new), 1) + rng.choice([0, 5])
        lens = [rng.randint(max(n, 1), most) if rng.random() < 0.7 else most for n in new]
        plans = [plan(rows, n, length, hq, hkv, window) for n, length in zip(new, lens) if n]
        wide = sum(p[1] for p in plans if not p[0])
        narrow = sum(p[1] for p in plans if p[0])
        parts = (wide * 128 + narrow * 32) * 130 * 4
        counts = 4 * (sum(p[2] for p in plans) + 17 * 32)
        need = lib.nc_packed_workspace_bytes(rows, batch, hq, hkv, most, window)
        assert parts <= need - need // 256 and counts <= need // 256, (hq, hkv, new, lens, window)


def sample_args(**over):
    args = dict(logits=DUMMY, is_bf16=0, row_stride=100, rows=4, vocab=100, uniform=DUMMY, temperature=DUMMY, top_k=None,
                top_p=None, min_p=None, mask=None, mask_stride=0, tokens=DUMMY, workspace=DUMMY, workspace_bytes=1 << 26, stream=None)
    return list((args | over).values())


def test_sample_rejects(lib):
    for name in ("logits", "uniform", "temperature", "tokens", "workspace"):
        assert lib.nc_sample_tokens(*sample_args(**{name: None})) == -1, name
    for over in (dict(rows=-1), dict(rows=2 ** 22 + 1), dict(vocab=0), dict(vocab=2 ** 24 + 1, row_stride=2 ** 25),
                 dict(row_stride=99), dict(mask=DUMMY, mask_stride=3), dict(workspace=ctypes.c_void_p(0x1008)), dict(workspace_bytes=15),
                 dict(vocab=8193, row_stride=8193, workspace_bytes=lib.nc_sample_workspace_bytes(4, 8193) - 1)):
        assert lib.nc_sample_tokens(*sample_args(**over)) == -2, over
    for rows, vocab in ((-1, 8), (2 ** 22 + 1, 8), (1, 0), (1, 2 ** 24 + 1)):
        assert lib.nc_sample_workspace_bytes(rows, vocab) == 0
    assert max(lib.nc_sample_workspace_bytes(2 ** 22, v) for v in (8192, 8193, 16385, 50257, 2 ** 18, 2 ** 18 + 1)) == 16
    most = max(lib.nc_sample_workspace_bytes(512 // g, 8192 * g) for g in range(2, 33))
    assert 6e6 < most < 7e6
    assert lib.nc_sample_tokens(*sample_args(rows=0)) == 0


@pytest.mark.parametrize("sizes", [(0, 4, 8), (4097, 4, 8), (4, 0, 8), (4, 4, 0), (4, 2 ** 27, 8), (4, 4, 2 ** 27)])
def test_block_tables_reject_sizes(sizes):
    with pytest.raises(ValueError):
        BlockTables(*sizes, "cpu")


def test_block_tables_need_a_device():
    with pytest.raises(ValueError, match="device tensor"):
        BlockTables(2, 2, 4, "cpu")
