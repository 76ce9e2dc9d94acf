"""Sizes of packed attention's Python entry points that do not fit the C ABI's 32-bit arguments."""
import pytest

from nanochat_amd.attention import packed_workspace_bytes


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1, 10 ** 30])
def test_a_window_past_every_position_hides_nothing(lib, window):
    """ctypes passes an integer's low 32 bits: 2^32 + 5 would be a window of 5 keys."""
    assert packed_workspace_bytes(64, 64, 16, 4, 40000, window) == packed_workspace_bytes(64, 64, 16, 4, 40000, -1)
    assert packed_workspace_bytes(64, 64, 16, 4, 40000, -window) == packed_workspace_bytes(64, 64, 16, 4, 40000, -1)


def test_a_misaligned_workspace_is_refused(lib):
    """Its partials are moved by 16-byte accesses."""
    import ctypes

    dummy = ctypes.c_void_p(0x1000)   # never dereferenced
    for at in (0x1001, 0x1004, 0x1008):
        assert lib.nc_packed_attn_fp8(dummy, dummy, dummy, dummy, dummy, 16, 8, dummy, dummy, 4, 2, 16, 4, 256, -1, 0.1, dummy,
                                      ctypes.c_void_p(at), 1 << 30, None) == -3, at


def test_more_sequences_than_a_launch_need_the_largest_launchs_workspace(lib):
    for rows, length in ((4096, 64), (20000, 40000)):
        most = packed_workspace_bytes(rows, 1024, 16, 4, length)
        assert most > 0
        for batch in (1025, 2000, 4096):
            assert packed_workspace_bytes(rows, batch, 16, 4, length) == most
        assert all(packed_workspace_bytes(rows, batch, 16, 4, length) <= most for batch in (1, 7, 100, 976))
