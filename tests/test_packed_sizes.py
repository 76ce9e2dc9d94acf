"""Sizes of packed attention's Python entry points that do not fit the C ABI's 32-bit arguments."""
import pytest

from nanochat_amd.attention import packed_workspace_bytes


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1, 10 ** 30])
def test_a_window_past_every_position_hides_nothing(lib, window):
    """ctypes passes an integer's low 32 bits: 2^32 + 5 would be a window of 5 keys."""
    assert packed_workspace_bytes(64, 64, 16, 4, 40000, window) == packed_workspace_bytes(64, 64, 16, 4, 40000, -1)
    assert packed_workspace_bytes(64, 64, 16, 4, 40000, -window) == packed_workspace_bytes(64, 64, 16, 4, 40000, -1)
