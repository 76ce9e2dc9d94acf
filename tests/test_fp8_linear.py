"""The 8-bit linear layers without a GPU: the registered ops and the shapes of their fake implementations, the wiring of their
gradients, and what the C ABI and the Python entry points refuse before any device call."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from nanochat_amd import fp8_linear as fl

DUMMY = ctypes.c_void_p(0x1000)   # never dereferenced: every call below fails its host checks first
CODES, SCALE, BF16, F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.float32


def held(n, k, d="cuda"):
    pad = lambda v: -(-(-(-v // 128)) // 4) * 4   # noqa: E731
    return (torch.empty(n, k, dtype=CODES, device=d), torch.empty(-(-n // 128), pad(k), dtype=SCALE, device=d),
            torch.empty(k, n, dtype=CODES, device=d), torch.empty(-(-k // 128), pad(n), dtype=SCALE, device=d))


@pytest.mark.parametrize("given", [False, True])
def test_fake_linear(given):
    with FakeTensorMode():
        x, w = torch.empty(2, 5, 400, dtype=BF16, device="cuda"), torch.empty(272, 400, device="cuda")
        out = torch.ops.nanochat_amd.checkpointed_linear(x, w, *(held(272, 400) if given else (None,) * 4), None)
        assert [(tuple(t.shape), t.dtype) for t in out[:3]] == [((2, 5, 272), BF16), ((10, 400), CODES), ((10, 4), SCALE)]
        assert [tuple(t.shape) for t in out[3:]] == ([(0,), (0,)] if given else [(400, 272), (4, 4)])
        _, _, ct, st = held(272, 400)
        for need_x, need_w, wide in ((True, True, True), (False, True, False), (True, False, True)):
            dx, dw = torch.ops.nanochat_amd.checkpointed_linear_bwd(out[0], out[1], out[2], ct, st, None, need_x, need_w, wide)
            assert tuple(dx.shape) == ((10, 400) if need_x else (0,))
            assert tuple(dw.shape) == ((272, 400) if need_w else (0,)) and (not need_w or dw.dtype == (F32 if wide else BF16))


def test_fake_mlp():
    with FakeTensorMode():
        x, fc, proj = (torch.empty(*s, dtype=BF16, device="cuda") for s in ((7, 256), (640, 256), (128, 640)))
        out = torch.ops.nanochat_amd.checkpointed_mlp(x, fc, proj, *(None,) * 5, *held(128, 640), None)
        assert [tuple(t.shape) for t in out] == [(7, 128), (7, 256), (7, 4), (7, 640), (7, 8), (256, 640), (2, 8), (0,), (0,)]
        _, _, pt, pts = held(128, 640)
        got = torch.ops.nanochat_amd.checkpointed_mlp_bwd(out[0], *out[1:7], pt, pts, None, torch.empty(128, 640, device="cuda"),
                                                          True, True, True, False, True)
        assert [tuple(t.shape) for t in got] == [(7, 256), (640, 256), (0,)]


def test_gradients_reach_their_inputs():
    """On meta tensors: x and the weights get gradients of their shapes; a weight with a buffer gets none."""
    x = torch.empty(3, 6, 256, dtype=BF16, device="meta", requires_grad=True)
    fc, proj = (torch.empty(*s, device="meta", requires_grad=True) for s in ((512, 256), (256, 512)))
    for buf in (None, torch.empty(512, 256, device="meta")):
        y = fl.checkpointed_mlp(fl.checkpointed_linear(x, torch.empty(256, 256, device="meta")), fc, proj, fc_grad=buf)
        got = torch.autograd.grad(y.float().sum(), (x, fc, proj), allow_unused=True)
        assert got[0].shape == x.shape and got[0].dtype == BF16 and got[2].shape == proj.shape and got[2].dtype == F32
        assert (got[1] is None) if buf is not None else got[1].shape == fc.shape


def test_gradients_have_no_gradient():
    x = torch.empty(4, 128, dtype=BF16, device="meta", requires_grad=True)
    w = torch.empty(128, 128, device="meta", requires_grad=True)
    for y in (fl.checkpointed_linear(x, w), fl.checkpointed_mlp(x, w, w)):
        dx, = torch.autograd.grad(y.float().pow(2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            dx.float().sum().backward()


def rows_args(**over):
    return list((dict(x=DUMMY, f32=0, stride=256, rows=3, cols=256, codes=DUMMY, scale=DUMMY, pitch=4, stream=None) | over).values())


def weight_args(**over):
    return list((dict(w=DUMMY, f32=0, stride=256, n=32, k=256, codes=DUMMY, scale=DUMMY, pitch=4, codes_t=DUMMY, scale_t=DUMMY,
                      pitch_t=4, stream=None) | over).values())


def product_args(**over):
    return dict(a=DUMMY, a_scale=DUMMY, a_pitch=4, w=DUMMY, w_scale=DUMMY, w_pitch=4, rows=3, n=32, k=256) | over


def grad_args(**over):
    return list((dict(dy=DUMMY, codes=DUMMY, scale=DUMMY, pitch=4, rows=3, n1=32, n2=256, mode=0, out=DUMMY, ws=DUMMY, bytes=16,
                      stream=None) | over).values())


def test_quantizers_refuse(lib):
    for name in ("x", "codes", "scale"):
        assert lib.nc_fp8_quantize_rows(*rows_args(**{name: None})) == -1, name
    for over in (dict(rows=-1), dict(cols=0), dict(cols=24), dict(cols=2 ** 20 + 16), dict(stride=255), dict(pitch=1),
                 dict(pitch=6), dict(rows=2 ** 30), dict(codes=ctypes.c_void_p(0x1008)), dict(scale=ctypes.c_void_p(0x1002)),
                 dict(x=ctypes.c_void_p(0x1001)), dict(x=ctypes.c_void_p(0x1002), f32=1)):
        assert lib.nc_fp8_quantize_rows(*rows_args(**over)) == -2, over
    assert lib.nc_fp8_quantize_rows(*rows_args(rows=0)) == 0
    for name in ("w", "codes", "scale", "scale_t"):
        assert lib.nc_fp8_quantize_weight(*weight_args(**{name: None})) == -1, name
    for over in (dict(n=0), dict(k=0), dict(k=250), dict(n=40), dict(n=2 ** 20 + 16), dict(stride=128), dict(pitch=1),
                 dict(pitch_t=0), dict(pitch_t=2), dict(codes_t=ctypes.c_void_p(0x1008))):
        assert lib.nc_fp8_quantize_weight(*weight_args(**over)) == -2, over


def test_products_refuse(lib):
    def all_three(over, status):
        args = list(product_args(**over).values())
        assert lib.nc_fp8_matmul(*args, DUMMY, None) == status, over
        assert lib.nc_fp8_matmul_relu2(*args, DUMMY, DUMMY, 4, None) == status, over
        assert lib.nc_fp8_matmul_relu2_bwd(*args, DUMMY, DUMMY, 4, DUMMY, DUMMY, DUMMY, 4, None) == status, over

    for name in ("a", "a_scale", "w", "w_scale"):
        all_three({name: None}, -1)
    for over in (dict(rows=-1), dict(n=0), dict(n=40), dict(k=0), dict(k=72), dict(n=2 ** 20 + 16), dict(a_pitch=1),
                 dict(a_pitch=6), dict(w_pitch=0), dict(a=ctypes.c_void_p(0x1008)), dict(w_scale=ctypes.c_void_p(0x1001))):
        all_three(over, -2)
    all_three(dict(rows=0), 0)
    args = list(product_args().values())
    assert lib.nc_fp8_matmul(*args, None, None) == -1
    for i in range(3):
        out = [DUMMY, DUMMY, 4]
        out[i] = None if i < 2 else 2
        assert lib.nc_fp8_matmul_relu2(*args, *out, None) == (-1 if i < 2 else -2)
    for i, bad in ((0, -1), (1, -1), (2, -2), (3, -1), (4, -1), (5, -1), (6, -2)):
        rest = [DUMMY, DUMMY, 4, DUMMY, DUMMY, DUMMY, 4]
        rest[i] = None if bad == -1 else 2
        assert lib.nc_fp8_matmul_relu2_bwd(*args, *rest, None) == bad, i


def linear_args(**over):
    return list((dict(x=DUMMY, f32=0, stride=256, w=DUMMY, w_scale=DUMMY, w_pitch=4, rows=80, n=32, k=256, out=DUMMY, ws=DUMMY,
                      bytes=2 ** 20, stream=None) | over).values())


def mlp_args(**over):
    return list((dict(x=DUMMY, stride=256, fc=DUMMY, fc_scale=DUMMY, fc_pitch=4, proj=DUMMY, proj_scale=DUMMY, proj_pitch=4, rows=40,
                      c=256, hidden=512, n=32, out=DUMMY, ws=DUMMY, bytes=2 ** 20, stream=None) | over).values())


def test_serving_refuses(lib):
    for name in ("x", "w", "w_scale", "out", "ws"):
        assert lib.nc_fp8_linear(*linear_args(**{name: None})) == -1, name
    odd = ctypes.c_void_p(0x1008)
    for over in (dict(rows=-1), dict(n=0), dict(n=40), dict(k=0), dict(k=72), dict(n=2 ** 20 + 16), dict(k=2 ** 20 + 16),
                 dict(rows=2 ** 30), dict(stride=255), dict(w_pitch=1), dict(w_pitch=6), dict(w=odd), dict(out=odd),
                 dict(x=ctypes.c_void_p(0x1001)), dict(x=ctypes.c_void_p(0x1002), f32=1)):
        assert lib.nc_fp8_linear(*linear_args(**over)) == -2, over
    need = lib.nc_fp8_linear_workspace_bytes(DUMMY, 0, 256, 80, 32, 256)
    assert need >= 80 * 256 + 80 * 2 and lib.nc_fp8_linear(*linear_args(bytes=need - 1)) == -3
    assert lib.nc_fp8_linear(*linear_args(ws=odd)) == -3 and lib.nc_fp8_linear(*linear_args(rows=0)) == 0
    for few in (dict(x=odd, ws=None), dict(rows=16, stride=257, ws=None), dict(rows=9, f32=1, ws=None),
                dict(n=2 ** 20, ws=None),
                dict(rows=65, ws=None), dict(rows=64, k=1296, stride=1296, w_pitch=12, ws=None)):   # these need it
        assert lib.nc_fp8_linear(*linear_args(**(dict(rows=2) | few))) == -1, few
    assert lib.nc_fp8_linear_workspace_bytes(DUMMY, 0, 24, 1, 16, 24) == -1
    assert lib.nc_fp8_linear_workspace_bytes(DUMMY, 0, 16, -1, 16, 16) == -1
    assert lib.nc_fp8_linear_workspace_bytes(DUMMY, 0, 256, 16, 32, 256) == 0
    assert lib.nc_fp8_linear_workspace_bytes(DUMMY, 0, 1280, 64, 32, 1280) == 0
    for name in ("x", "fc", "fc_scale", "proj", "proj_scale", "out", "ws"):
        assert lib.nc_fp8_mlp(*mlp_args(**{name: None})) == -1, name
    for over in (dict(rows=-1), dict(c=0), dict(c=40), dict(hidden=500), dict(n=20), dict(hidden=2 ** 20 + 16), dict(stride=255),
                 dict(fc_pitch=1), dict(proj_pitch=2), dict(fc=odd), dict(proj=odd), dict(out=odd)):
        assert lib.nc_fp8_mlp(*mlp_args(**over)) == -2, over
    need = lib.nc_fp8_mlp_workspace_bytes(40, 256, 512)
    assert lib.nc_fp8_mlp(*mlp_args(bytes=need - 1)) == -3 and lib.nc_fp8_mlp(*mlp_args(ws=odd)) == -3
    assert lib.nc_fp8_mlp(*mlp_args(rows=0)) == 0 and lib.nc_fp8_mlp_workspace_bytes(40, 256, 500) == -1


def test_training_refuses(lib):
    def fwd(**over):
        a = dict(x=DUMMY, stride=256, w=DUMMY, w_scale=DUMMY, w_pitch=4, rows=3, n=32, k=256, codes=DUMMY, scale=DUMMY, pitch=4,
                 out=DUMMY, stream=None) | over
        return lib.nc_fp8_linear_fwd(*a.values())

    def bwd(**over):
        a = dict(dy=DUMMY, stride=32, codes=DUMMY, scale=DUMMY, pitch=4, codes_t=DUMMY, scale_t=DUMMY, pitch_t=4, rows=3, n=32,
                 k=256, dx=DUMMY, dw=DUMMY, mode=0, ws=DUMMY, bytes=2 ** 20, stream=None) | over
        return lib.nc_fp8_linear_bwd(*a.values())

    def mlp_fwd(**over):
        a = dict(x=DUMMY, stride=256, fc=DUMMY, fc_scale=DUMMY, fc_pitch=4, proj=DUMMY, proj_scale=DUMMY, proj_pitch=4, rows=3,
                 c=256, hidden=512, n=32, codes=DUMMY, scale=DUMMY, pitch=4, act=DUMMY, act_scale=DUMMY, act_pitch=4, out=DUMMY,
                 stream=None) | over
        return lib.nc_fp8_mlp_fwd(*a.values())

    def mlp_bwd(**over):
        a = dict(dy=DUMMY, stride=32, codes=DUMMY, scale=DUMMY, pitch=4, act=DUMMY, act_scale=DUMMY, act_pitch=4, fct=DUMMY,
                 fct_scale=DUMMY, fct_pitch=4, pt=DUMMY, pt_scale=DUMMY, pt_pitch=4, rows=3, c=256, hidden=512, n=32, dx=DUMMY,
                 dfc=DUMMY, fc_mode=0, dproj=DUMMY, proj_mode=0, ws=DUMMY, bytes=2 ** 24, stream=None) | over
        return lib.nc_fp8_mlp_bwd(*a.values())

    odd = ctypes.c_void_p(0x1008)
    for call, names in ((fwd, ("x", "w", "w_scale", "codes", "scale", "out")),
                        (bwd, ("dy", "codes", "scale", "codes_t", "scale_t", "dw", "ws")),
                        (mlp_fwd, ("x", "fc", "fc_scale", "proj", "proj_scale", "codes", "scale", "act", "act_scale", "out")),
                        (mlp_bwd, ("dy", "codes", "scale", "act", "act_scale", "fct", "fct_scale", "pt", "pt_scale", "dfc",
                                   "dproj", "ws"))):
        for name in names:
            assert call(**{name: None}) == -1, (call, name)
        for over in (dict(rows=-1), dict(n=24), dict(n=0)):
            assert call(**over) == -2, (call, over)
        assert call(rows=0) == 0
    assert fwd(k=72) == fwd(w=odd) == fwd(out=odd) == fwd(pitch=1) == mlp_fwd(hidden=500) == mlp_fwd(act=odd) == -2
    assert bwd(mode=3) == bwd(stride=40) == mlp_bwd(fc_mode=-2) == mlp_bwd(stride=40) == mlp_bwd(c=2 ** 20 + 16) == -2
    need = lib.nc_fp8_linear_bwd_workspace_bytes(3, 32, 256, 1, 0)
    assert bwd(bytes=need - 1) == bwd(ws=odd) == -3
    need = lib.nc_fp8_mlp_bwd_workspace_bytes(3, 256, 512, 32, 1, 0, 0)
    assert mlp_bwd(bytes=need - 1) == mlp_bwd(ws=odd) == -3
    assert lib.nc_fp8_linear_bwd_workspace_bytes(3, 32, 256, 0, -1) == 0 == lib.nc_fp8_mlp_bwd_workspace_bytes(3, 256, 512, 32, 0, -1, -1)


def test_weight_gradient_refuses(lib):
    for name in ("dy", "codes", "scale", "out", "ws"):
        assert lib.nc_fp8_weight_grad(*grad_args(**{name: None})) == -1, name
    for over in (dict(rows=-1), dict(n1=4), dict(n2=24), dict(n1=65536 + 8), dict(mode=3), dict(mode=-1), dict(pitch=1),
                 dict(pitch=512), dict(out=ctypes.c_void_p(0x1008)), dict(rows=2 ** 31)):
        assert lib.nc_fp8_weight_grad(*grad_args(**over)) == -2, over
    need = lib.nc_fp8_weight_grad_workspace_bytes(4096, 256, 256)
    assert need > 16 and lib.nc_fp8_weight_grad(*grad_args(rows=4096, n1=256, bytes=need - 1)) == -3
    assert lib.nc_fp8_weight_grad_workspace_bytes(1, 4, 16) == -1 and lib.nc_fp8_weight_grad(*grad_args(rows=0)) == 0


def test_entry_points_need_device_tensors():
    x, w = torch.zeros(4, 128, dtype=BF16), torch.zeros(32, 128)
    codes, scale = torch.zeros(4, 128).to(CODES), torch.zeros(4, 4, dtype=torch.uint8).view(SCALE)[:, :1]
    w8 = fl.Fp8Weight(torch.zeros(32, 128).to(CODES), scale[:1])
    for call in (lambda: fl.quantize_rows(x), lambda: fl.quantize_weight(w), lambda: fl.fp8_linear(x, w8),
                 lambda: fl.fp8_mlp(x, w8, w8), lambda: fl.fp8_matmul(codes, scale, w8),
                 lambda: fl.checkpoint_weight_grad(x, codes, scale)):
        with pytest.raises(ValueError, match="device tensor"):
            call()
