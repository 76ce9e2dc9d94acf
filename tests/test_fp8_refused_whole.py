"""The C calls of the 8-bit layers refuse what any of their kernels cannot take, before the first launch: a call that is refused has
written nothing. Without a GPU a launch gives the runtime's own status, so a call that launched first shows."""
import ctypes

import pytest

DUMMY, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008)   # never dereferenced


@pytest.mark.parametrize("over", [dict(scale=ctypes.c_void_p(0x1002)), dict(pitch=5), dict(pitch=6)])
def test_weight_gradient_takes_whole_dwords_of_scales(lib, over):
    """They are fetched four at a time."""
    a = dict(dy=DUMMY, codes=DUMMY, scale=DUMMY, pitch=4, rows=3, n1=32, n2=256, mode=0, out=DUMMY, ws=DUMMY, bytes=16, stream=None)
    assert lib.nc_fp8_weight_grad(*(a | over).values()) == -2
