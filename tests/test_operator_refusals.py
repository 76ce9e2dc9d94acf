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


def sample_args(**over):
    args = dict(logits=DUMMY, is_bf16=0, row_stride=100, rows=4, vocab=100, uniform=DUMMY, temperature=DUMMY, top_k=None,
                top_p=None, min_p=None, mask=None, mask_stride=0, tokens=DUMMY, stream=None)
    return list((args | over).values())


def test_sample_rejects(lib):
    for name in ("logits", "uniform", "temperature", "tokens"):
        assert lib.nc_sample_tokens(*sample_args(**{name: None})) == -1, name
    for over in (dict(rows=-1), dict(rows=2 ** 22 + 1), dict(vocab=0), dict(vocab=2 ** 24 + 1, row_stride=2 ** 25),
                 dict(row_stride=99), dict(mask=DUMMY, mask_stride=3)):
        assert lib.nc_sample_tokens(*sample_args(**over)) == -2, over
    assert lib.nc_sample_tokens(*sample_args(rows=0)) == 0


@pytest.mark.parametrize("sizes", [(0, 4, 8), (4097, 4, 8), (4, 0, 8), (4, 4, 0), (4, 2 ** 27, 8), (4, 4, 2 ** 27)])
def test_block_tables_reject_sizes(sizes):
    with pytest.raises(ValueError):
        BlockTables(*sizes, "cpu")


def test_block_tables_need_a_device():
    with pytest.raises(ValueError, match="device tensor"):
        BlockTables(2, 2, 4, "cpu")
