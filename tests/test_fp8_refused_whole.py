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


FORMS = {"linear_fwd": [("w", "w_scale", "w_pitch"), ("codes", "scale", "pitch")],
         "linear_bwd": [("codes", "scale", "pitch"), ("codes_t", "scale_t", "pitch_t")],
         "mlp_fwd": [("fc", "fc_scale", "fc_pitch"), ("proj", "proj_scale", "proj_pitch"), ("codes", "scale", "pitch"),
                     ("act", "act_scale", "act_pitch")],
         "mlp_bwd": [("codes", "scale", "pitch"), ("act", "act_scale", "act_pitch"), ("fct", "fct_scale", "fct_pitch"),
                     ("pt", "pt_scale", "pt_pitch")]}
ARGS = {
    "linear_fwd": dict(x=DUMMY, stride=256, w=DUMMY, w_scale=DUMMY, w_pitch=4, rows=3, n=32, k=256, codes=DUMMY, scale=DUMMY, pitch=4,
                       out=DUMMY, stream=None),
    "linear_bwd": dict(dy=DUMMY, stride=32, codes=DUMMY, scale=DUMMY, pitch=4, codes_t=DUMMY, scale_t=DUMMY, pitch_t=4, rows=3, n=32,
                       k=256, dx=DUMMY, dw=DUMMY, mode=0, ws=DUMMY, bytes=2 ** 20, stream=None),
    "mlp_fwd": dict(x=DUMMY, stride=256, fc=DUMMY, fc_scale=DUMMY, fc_pitch=4, proj=DUMMY, proj_scale=DUMMY, proj_pitch=4, rows=3,
                    c=256, hidden=512, n=32, codes=DUMMY, scale=DUMMY, pitch=4, act=DUMMY, act_scale=DUMMY, act_pitch=4, out=DUMMY,
                    stream=None),
    "mlp_bwd": dict(dy=DUMMY, stride=32, codes=DUMMY, scale=DUMMY, pitch=4, act=DUMMY, act_scale=DUMMY, act_pitch=4, fct=DUMMY,
                    fct_scale=DUMMY, fct_pitch=4, pt=DUMMY, pt_scale=DUMMY, pt_pitch=4, rows=3, c=256, hidden=512, n=32, dx=DUMMY,
                    dfc=DUMMY, fc_mode=0, dproj=DUMMY, proj_mode=0, ws=DUMMY, bytes=2 ** 24, stream=None)}
OUTPUTS = {"linear_fwd": ["out"], "linear_bwd": ["dx", "dw"], "mlp_fwd": ["out"], "mlp_bwd": ["dx", "dfc", "dproj"]}


def status(lib, name, **over):
    assert not over.keys() - ARGS[name].keys()
    return getattr(lib, f"nc_fp8_{name}")(*(ARGS[name] | over).values())


@pytest.mark.parametrize("name", ARGS)
def test_forms_and_outputs(lib, name):
    for codes, scale, pitch in FORMS[name]:
        for over in ({codes: ODD}, {scale: ctypes.c_void_p(0x1002)}, {pitch: 0}, {pitch: 6}, {pitch: 2 ** 14 + 4}):
            assert status(lib, name, **over) == -2, over
    for out in OUTPUTS[name]:
        assert status(lib, name, **{out: ODD}) == -2, out


def test_rows(lib):
    for name in ("linear_fwd", "mlp_fwd"):
        for over in (dict(x=ctypes.c_void_p(0x1001)), dict(stride=255), dict(stride=2 ** 41)):
            assert status(lib, name, **over) == -2, over
    for name in ("linear_bwd", "mlp_bwd"):
        off = dict(mode=-1) if name == "linear_bwd" else dict(proj_mode=-1)
        for over in (dict(dy=ODD), dict(dy=ctypes.c_void_p(0x1001), **off), dict(stride=31, **off), dict(stride=2 ** 41, **off)):
            assert status(lib, name, **over) == -2, over


def test_what_is_not_read_is_not_refused(lib):
    """rows = 0 reads nothing; without a gradient its operands may be missing."""
    for name in ARGS:
        assert status(lib, name, rows=0, **{codes: ODD for codes, _, _ in FORMS[name]}) == 0, name
    none = dict(rows=0, dx=None)
    assert status(lib, "linear_bwd", mode=-1, dw=None, codes=None, codes_t=None, **none) == 0
    assert status(lib, "mlp_bwd", fc_mode=-1, proj_mode=-1, dfc=None, dproj=None, codes=None, fct=None, pt=None, **none) == 0
