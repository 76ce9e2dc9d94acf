"""What the 8-bit layers hand to the library, without a GPU: host tensors that say they lie on a device, and a library that
records its calls. Operands that do not belong together have to be refused before any of them."""
import contextlib

import pytest
import torch

from nanochat_amd import fp8_linear as fl, native

CODES, SCALE, BF16, F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.float32


class OnDevice(torch.Tensor):
    is_cuda = True


class Recorder:
    """The library's functions by name: calls of theirs are kept, and answered from `answers` (else 0)."""

    def __init__(self):
        self.calls, self.answers = [], {}

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return self.answers.get(name, 0)
        return call

    def named(self, name):
        return [args for n, args in self.calls if n == name]


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(fl, "hip_library", lambda: r)
    monkeypatch.setattr(native, "hip_library", lambda: native_strings)
    monkeypatch.setattr(fl, "device_guard", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(fl, "stream", lambda: 0)
    return r


class native_strings:
    @staticmethod
    def nc_status_string(status):
        return b"a status"


def new(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=torch.uint8).view(dtype).as_subclass(OnDevice) if dtype in (CODES, SCALE) else \
        torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


def up4(n):
    return -(-n // 4) * 4


def form(rows, cols, of=1, whole=True):
    blocks = -(-cols // 128)
    scale = new(-(-rows // of), up4(blocks), dtype=SCALE)
    return new(rows, cols, dtype=CODES), scale if whole else scale[:, :blocks]


# --- the backward ops, given operands that do not belong together

M, N, K, F = 10, 528, 656, 560   # of more blocks than one dword of scales holds


def linear_bwd(**over):
    x8, xs = form(M, K)
    codes_t, scale_t = form(K, N, 128)
    a = dict(dy=new(M, N), x8=x8, xs=xs, codes_t=codes_t, scale_t=scale_t, grad=None, need_x=True, need_w=True, wide=True) | over
    return fl._run_linear_bwd(**a)


def mlp_bwd(**over):
    """x [M, K], fc [F, K], proj [N, F]"""
    x8, xs = form(M, K)
    a8, a_s = form(M, F)
    f, fs = form(K, F, 128)
    p, ps = form(F, N, 128)
    a = dict(dy=new(M, N), x8=x8, xs=xs, a8=a8, a_s=a_s, fc_codes_t=f, fc_scale_t=fs, proj_codes_t=p, proj_scale_t=ps, fc_grad=None,
             proj_grad=None, need_x=True, need_fc=True, need_proj=True, fc_wide=True, proj_wide=True) | over
    return fl._run_mlp_bwd(**a)


WRONG_FORMS = {"fewer rows": lambda r, c, of: form(r - of, c, of), "more rows": lambda r, c, of: form(r + of, c, of),
               "fewer columns": lambda r, c, of: form(r, 16, of), "no tensor of the op": lambda r, c, of: form(0, 16, of)}
LINEAR_FORMS = {"x8": ("xs", M, K, 1), "codes_t": ("scale_t", K, N, 128)}
MLP_FORMS = {"x8": ("xs", M, K, 1), "a8": ("a_s", M, F, 1), "fc_codes_t": ("fc_scale_t", K, F, 128),
             "proj_codes_t": ("proj_scale_t", F, N, 128)}
BOTH = [(linear_bwd, name, *v) for name, v in LINEAR_FORMS.items()] + [(mlp_bwd, name, *v) for name, v in MLP_FORMS.items()]


@pytest.mark.parametrize("call,codes,scale,rows,cols,of", BOTH)
@pytest.mark.parametrize("wrong", WRONG_FORMS)
def test_backward_ops_refuse_forms_of_other_sizes(recorder, call, codes, scale, rows, cols, of, wrong):
    c, s = WRONG_FORMS[wrong](rows, cols, of)
    right_c, right_s = form(rows, cols, of)
    for over in ({codes: c, scale: s}, {codes: right_c, scale: s}, {codes: c, scale: right_s}):
        with pytest.raises(ValueError):
            call(**over)
    assert not recorder.calls


@pytest.mark.parametrize("call,codes,scale,rows,cols,of", BOTH)
def test_backward_ops_refuse_forms_of_other_types_and_places(recorder, call, codes, scale, rows, cols, of):
    c, s = form(rows, cols, of)
    for over in ({codes: c.float()}, {codes: c.view(torch.uint8)}, {scale: s.view(torch.uint8)}, {scale: s.float()}):
        with pytest.raises(TypeError):
            call(**over)
    for over in ({codes: c.as_subclass(torch.Tensor)}, {codes: c.as_subclass(torch.Tensor).to("meta")},
                 {scale: s.as_subclass(torch.Tensor).to("meta")}, {codes: form(cols, rows // 16 * 16 + 16, of)[0].t()[:rows]},
                 {scale: s.repeat(1, 3)[:, :s.size(1)][:, ::1].t().contiguous().t()}):
        with pytest.raises(ValueError):
            call(**over)
    assert not recorder.calls


def test_backward_ops_take_forms_with_and_without_padding(recorder):
    """As the forward ops return them, and as quantize_weight does; what a call does not read it does not check."""
    for whole in (True, False):
        linear_bwd(**dict(zip(("x8", "xs"), form(M, K, whole=whole))), **dict(zip(("codes_t", "scale_t"), form(K, N, 128, whole))))
        mlp_bwd(**dict(zip(("a8", "a_s"), form(M, F, whole=whole))),
                **dict(zip(("proj_codes_t", "proj_scale_t"), form(F, N, 128, whole))))
    empty = new(0, dtype=CODES), new(0, dtype=SCALE)
    linear_bwd(codes_t=empty[0], scale_t=empty[1], need_x=False)
    mlp_bwd(fc_codes_t=empty[0], fc_scale_t=empty[1], need_x=False)
    mlp_bwd(fc_codes_t=empty[0], fc_scale_t=empty[1], proj_codes_t=empty[0], proj_scale_t=empty[1], need_x=False, need_fc=False)
    assert len(recorder.named("nc_fp8_linear_bwd")) == 3 and len(recorder.named("nc_fp8_mlp_bwd")) == 4
    assert all(args[8:11] == (M, N, K) for args in recorder.named("nc_fp8_linear_bwd"))


# --- gradient buffers, where they are written

def bad_buffers(n, k):
    return [new(n, k, dtype=torch.float64), new(n, k), new(16, 16, dtype=F32), new(k, n, dtype=F32), new(n * k, dtype=F32),
            new(k, n, dtype=F32).t(), new(n, 2 * k, dtype=F32)[:, :k], new(n * k + 1, dtype=F32)[1:].view(n, k),
            torch.zeros(n, k, device="meta")]


def test_backward_ops_refuse_buffers_that_do_not_fit(recorder):
    for call, name, n, k in ((linear_bwd, "grad", N, K), (mlp_bwd, "fc_grad", F, K), (mlp_bwd, "proj_grad", N, F)):
        for bad in bad_buffers(n, k):
            with pytest.raises(ValueError, match=name):
                call(**{name: bad})
        assert not recorder.calls
        call(**{name: new(n, k, dtype=F32)})
        assert len(recorder.named("nc_fp8_linear_bwd") + recorder.named("nc_fp8_mlp_bwd")) == 1
        recorder.calls.clear()


@pytest.mark.parametrize("other", [dict(dtype=torch.float64), dict(shape=(16, 16)), dict(dtype=BF16)])
def test_a_buffer_exchanged_before_the_backward_is_refused(recorder, monkeypatch, other):
    """The forward has checked it; what counts is what it is when it is added to."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)   # of what the calls make themselves too
    monkeypatch.setattr(fl, "_linear", fl._run_linear)
    monkeypatch.setattr(fl, "_linear_bwd", fl._run_linear_bwd)
    monkeypatch.setattr(fl, "_mlp", fl._run_mlp)
    monkeypatch.setattr(fl, "_mlp_bwd", fl._run_mlp_bwd)
    x = new(M, K).requires_grad_()
    for layer, shape in ((lambda b: fl.checkpointed_linear(x, new(N, K), grad=b), (N, K)),
                         (lambda b: fl.checkpointed_mlp(x, new(F, K), new(N, F), fc_grad=b), (F, K)),
                         (lambda b: fl.checkpointed_mlp(x, new(F, K), new(N, F), proj_grad=b), (N, F))):
        buffer = new(*shape, dtype=F32)
        y = layer(buffer)
        recorder.calls.clear()
        buffer.data = torch.zeros(other.get("shape", shape), dtype=other.get("dtype", F32))
        with pytest.raises(ValueError, match="grad must be"):
            y.backward(new(M, y.size(-1)))
        assert not recorder.calls


# --- statuses

@pytest.mark.parametrize("rows", [1, 40, 64])
@pytest.mark.parametrize("status", [-2, -3, 1, 98, 719])
def test_a_failed_launch_of_a_few_rows_is_reported(recorder, rows, status):
    """Only a missing workspace's status has the call made again with one: a failure's would be lost behind a second call that
    returns 0."""
    w8 = fl.Fp8Weight(*form(N, K, 128, whole=False))
    answers = iter([status])
    recorder.nc_fp8_linear = lambda *args: (recorder.calls.append(("nc_fp8_linear", args)), next(answers, 0))[1]
    with pytest.raises(native.NativeError, match=str(status)):
        fl.fp8_linear(new(rows, K), w8)
    assert len(recorder.named("nc_fp8_linear")) == 1


@pytest.mark.parametrize("second", [0, 98])
def test_a_missing_workspace_is_brought(recorder, second):
    w8 = fl.Fp8Weight(*form(N, K, 128, whole=False))
    answers = iter([-1, second])
    recorder.answers["nc_fp8_linear_workspace_bytes"] = 4096
    recorder.nc_fp8_linear = lambda *args: (recorder.calls.append(("nc_fp8_linear", args)), next(answers))[1]
    if second:
        with pytest.raises(native.NativeError, match="98"):
            fl.fp8_linear(new(40, K), w8)
    else:
        assert fl.fp8_linear(new(40, K), w8).shape == (40, N)
    without, given = recorder.named("nc_fp8_linear")
    assert without[10:12] == (None, 0) and given[10] is not None and given[11] == 4096


# --- autograd's bookkeeping

def test_a_weight_gradient_added_in_place_is_noticed(recorder):
    """A backward that needs the buffer as it was refuses to run on what it has become."""
    codes, scale = form(M, K, whole=False)
    out, factor = new(N, K, dtype=F32).as_subclass(torch.Tensor), torch.ones(N, K, requires_grad=True)
    y = (factor * out).sum()
    fl.checkpoint_weight_grad(new(M, N), codes, scale, out=out.as_subclass(OnDevice))
    assert len(recorder.named("nc_fp8_weight_grad")) == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():   # such tensors have no versions
        fl.checkpoint_weight_grad(new(M, N), codes, scale, out=new(N, K, dtype=F32))


@pytest.fixture
def eager(recorder, monkeypatch):
    """The ops' own functions in place of the dispatcher, which has none for host tensors."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    for name in ("linear", "linear_bwd", "mlp", "mlp_bwd"):
        monkeypatch.setattr(fl, f"_{name}", getattr(fl, f"_run_{name}"))
    return recorder


def test_a_buffer_is_added_to_whatever_requires_a_gradient(eager):
    """Frozen weights, or such as are no parameters, on inputs without a gradient: the first layer of a model that keeps its
    gradients in buffers."""
    x, w, f, p = new(M, K), new(N, K), new(F, K), new(N, F)
    buffer = lambda t: new(*t.shape, dtype=F32)   # noqa: E731
    for layer, name, modes in ((lambda: fl.checkpointed_linear(x, w, grad=buffer(w)), "linear", {13: 1}),
                               (lambda: fl.checkpointed_mlp(x, f, p, fc_grad=buffer(f)), "mlp", {20: 1, 22: -1}),
                               (lambda: fl.checkpointed_mlp(x, f, p, proj_grad=buffer(p)), "mlp", {20: -1, 22: 1}),
                               (lambda: fl.checkpointed_mlp(x, f, p, fc_grad=buffer(f), proj_grad=buffer(p)), "mlp", {20: 1, 22: 1})):
        y = layer()
        assert y.requires_grad
        y.backward(new(M, N))
        call, = eager.named(f"nc_fp8_{name}_bwd")
        assert {i: call[i] for i in modes} == modes and all(t.grad is None and not t.requires_grad for t in (x, w, f, p))
        eager.calls.clear()
        with torch.no_grad():
            assert not layer().requires_grad
    assert not fl.checkpointed_linear(x, w).requires_grad and not fl.checkpointed_mlp(x, f, p).requires_grad


def test_a_buffer_of_a_layer_that_is_recorded_anyway(eager):
    for x, w in ((new(M, K).requires_grad_(), new(N, K)), (new(M, K), new(N, K).requires_grad_())):
        y = fl.checkpointed_linear(x, w, grad=new(N, K, dtype=F32))
        y.backward(new(M, N))
        assert w.grad is None and (x.grad is not None) == x.requires_grad
    assert [args[13] for args in eager.named("nc_fp8_linear_bwd")] == [1, 1]


@pytest.mark.parametrize("asked", ["x", "weight", "nothing"])
def test_layers_trace_without_a_break(asked):
    """With a buffer, whatever requires a gradient (on meta tensors, through the ops' fakes)."""
    x = torch.empty(4, 256, dtype=BF16, device="meta", requires_grad=asked == "x")
    w, p = (torch.empty(*s, device="meta", requires_grad=asked == "weight") for s in ((128, 256), (256, 128)))

    def layers(x, buffer):
        return fl.checkpointed_mlp(x, w, p, fc_grad=buffer) + fl.checkpointed_mlp(x, w, p, proj_grad=buffer.t().contiguous(), fast=True)

    torch._dynamo.reset()
    y = torch.compile(layers, fullgraph=True, backend="aot_eager")(x, torch.empty(128, 256, device="meta"))
    assert y.requires_grad and y.shape == x.shape


def test_saved_tensors_that_hooks_lay_out_anew(eager):
    """Tensors kept for the backward may come back contiguous, as from host memory: the scales of a weight held by the caller, views
    of wider rows, then lack their padding."""
    def held(n, k):
        return fl.Fp8Weight(*form(n, k, 128, whole=False), *form(k, n, 128, whole=False))

    x = new(M, K).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t):
        y = fl.checkpointed_linear(x, new(N, K), held(N, K)), fl.checkpointed_mlp(x, new(F, K), new(N, F), held(F, K), held(N, F))
    for t in y:
        t.backward(new(M, N))
    linear, = eager.named("nc_fp8_linear_bwd")
    mlp, = eager.named("nc_fp8_mlp_bwd")
    assert linear[7] == 8 and (mlp[10], mlp[13]) == (8, 8)   # the pitches of 5 blocks
