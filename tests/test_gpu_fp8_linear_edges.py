"""More of the 8-bit linear layers on the GPU: calls that the documentation allows at the edges of what tests/test_gpu_fp8_linear.py
runs. Bounds as there."""
import numpy as np
import pytest
import torch

from nanochat_amd import fp8_linear as fl, native
from nanochat_amd.native import hip_library, stream
from oracle import fp8_block as fb
from tests import test_gpu_fp8_linear as whole
from tests.test_gpu_fp8_linear import EPS, SIZES, bf, close, codes_of, exps_of, form, held, product_relu2, product_relu2_bwd, same_form, weight

pytestmark = pytest.mark.gpu


def at_the_end(scale, wider):
    """The same scales as the last columns of wider rows, at the very end of their storage."""
    rows, blocks = scale.shape
    pad = -(-blocks // 4) * 4
    whole = torch.zeros(rows, pad + wider, dtype=torch.uint8, device=scale.device)
    whole[:, wider:wider + blocks] = scale.contiguous().view(torch.uint8)
    return whole.view(fl.SCALE)[:, wider:wider + blocks]


@pytest.mark.parametrize("rows,n,k", [(8, 528, 2048), (70, 1296, 512), (600, 4112, 512), (4100, 4112, 1024)])
def test_scales_that_end_with_their_storage(device, rows, n, k):
    """Few results, small, half and full tiles."""
    gen = torch.Generator().manual_seed(rows + k)
    codes, scale, _ = form(gen, device, rows, k)
    w, _ = weight(gen, device, n, k)
    want = fl.fp8_matmul(codes, scale, w)
    for wider in (4, 48):
        assert torch.equal(fl.fp8_matmul(codes, at_the_end(scale, wider), fl.Fp8Weight(w.codes, at_the_end(w.scale, wider))), want)
    dy = bf(gen, rows, 144).to(device)
    assert torch.equal(fl.checkpoint_weight_grad(dy, codes, at_the_end(scale, 48)), fl.checkpoint_weight_grad(dy, codes, scale))


def test_buffers_of_layers_without_a_gradient(device):
    """Neither the input nor the weights require one: what the buffers are given is what a parameter would get."""
    gen = torch.Generator().manual_seed(20)
    x, dy = bf(gen, 70, 256).to(device), bf(gen, 70, 144).to(device)
    w, fc, proj = (torch.randn(*s, generator=gen).to(device) / 16 for s in ((144, 256), (640, 256), (144, 640)))
    buffers = [torch.zeros_like(t) for t in (w, fc, proj)]
    fl.checkpointed_linear(x, w, grad=buffers[0]).backward(dy)
    fl.checkpointed_mlp(x, fc, proj, fc_grad=buffers[1], proj_grad=buffers[2]).backward(dy)
    asked = [t.clone().requires_grad_() for t in (w, fc, proj)]
    fl.checkpointed_linear(x, asked[0]).backward(dy)
    fl.checkpointed_mlp(x, *asked[1:]).backward(dy)
    # the same sums, added to zeros
    assert all(torch.equal(b, t.grad) for b, t in zip(buffers, asked)) and all(t.grad is None for t in (w, fc, proj))
    # captured, beside an eager call that has not been differentiated yet
    waiting = fl.checkpointed_linear(x, w, grad=torch.zeros_like(w))
    into, held_x, held_dy = [torch.zeros_like(t) for t in (w, fc, proj)], x.clone(), dy.clone()

    def step():
        for t in into:
            t.zero_()
        fl.checkpointed_linear(held_x, w, grad=into[0]).backward(held_dy)
        fl.checkpointed_mlp(held_x, fc, proj, fc_grad=into[1], proj_grad=into[2]).backward(held_dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        held_x.copy_(bf(gen, 70, 256).to(device))
        graph.replay()
        held_x.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(into, buffers))
    waiting.backward(dy)


@pytest.mark.parametrize("rows,n,k", [(8190, 4352, 768), (12000, 2832, 1152)])
def test_several_tiles_a_workgroup_write_nothing_else(device, rows, n, k):
    whole.test_products_write_their_results_and_nothing_else(device, rows, n, k)
    gen = torch.Generator().manual_seed(rows)
    codes, scale, _ = form(gen, device, rows, k)
    w, _ = weight(gen, device, n, k)
    a8, a_s = relu2_fast(codes, scale, w)
    out, exps = torch.full((rows + 600, n), 0xA5, dtype=torch.uint8, device=device), fl._new_scale(codes, rows, n)
    native.check(hip_library().nc_fp8_matmul_relu2_fast(codes.data_ptr(), scale.data_ptr(), scale.stride(0), w.codes.data_ptr(),
                                                        w.scale.data_ptr(), w.scale.stride(0), rows, n, k, out[300:].data_ptr(),
                                                        exps.data_ptr(), exps.stride(0), stream()))
    assert torch.equal(out[300:300 + rows], a8.view(torch.uint8))
    out[300:300 + rows] = 0xA5
    assert bool((out == 0xA5).all())


def relu2_fast(codes, scale, w):
    """product_relu2 by the products that drop bits in half and full tiles."""
    rows, k = codes.shape
    n = w.codes.size(0)
    out, out_scale = torch.empty(rows, n, dtype=fl.CODES, device=codes.device), fl._new_scale(codes, rows, n)
    native.check(hip_library().nc_fp8_matmul_relu2_fast(codes.data_ptr(), scale.data_ptr(), scale.stride(0), w.codes.data_ptr(),
                                                         w.scale.data_ptr(), w.scale.stride(0), rows, n, k, out.data_ptr(),
                                                         out_scale.data_ptr(), out_scale.stride(0), stream()))
    return out, out_scale


# --- long walks, and workgroups that take several tiles (256 CUs; stages of 128 columns)

# rows, outputs, columns: what the product's rule makes of them
LONG = [(65, 1280, 1168),       # small tiles before a ReLU^2, 10 stages
        (130, 8208, 1168),      # small tiles, 195
        (600, 4112, 1168),      # half tiles, 165, 10 stages
        (2500, 1680, 2000),     # half tiles, 16 stages
        (9300, 2064, 1168),     # full tiles, 252, and half ones; a last column of 16
        (6100, 5520, 640),      # 506 full tiles, two a workgroup, 5 stages; the last column of 144
        (12000, 2832, 1152),    # 504, 9 stages; the last column of 16: two of a tile's four waves have nothing
        (8400, 4112, 1664),     # 510, 13 stages; the same
        (8190, 4352, 768),      # 510, 6 stages
        (8190, 6144, 528),      # 768, three a workgroup, 5 stages, the last of 16 columns
        (8190, 6144, 256),      # 768 of 2 stages
        (8190, 6144, 128)]      # 768 of one


def uneven(gen, device, rows, cols, of):
    """Values whose blocks (of `of` rows and 128 columns) lie up to 2^6 apart, so that a wrong block's scale shows anywhere."""
    x = torch.randn(rows, cols, generator=gen)
    e = torch.randint(-3, 4, (-(-rows // of), -(-cols // 128)), generator=gen).float()
    return x * torch.exp2(e).repeat_interleave(of, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def sampled(rows):
    """Rows of every tile, at its waves' borders and at places of their own."""
    return [r for r in range(rows) if r % 64 in (0, 15, 16, 63) or r == rows - 1 or r % 61 == 7]


def operands(device, rows, n, k):
    gen = torch.Generator().manual_seed(rows + n + k)
    codes, scale = fl.quantize_rows(uneven(gen, device, rows, k, 1).to(torch.bfloat16).to(device))
    w = fl.quantize_weight((uneven(gen, device, n, k, 128) * k ** -0.5).to(device))
    at = sampled(rows)
    there = torch.tensor(at, device=device)
    x = fb.values(codes_of(codes[there].contiguous()), exps_of(scale[there]), 1)
    wv = fb.values(codes_of(w.codes), exps_of(w.scale), 128)
    return gen, codes, scale, w, there, x @ wv.T, (2.0 ** -10 + k * EPS) * (np.abs(x) @ np.abs(wv).T)


@pytest.mark.parametrize("rows,n,k", LONG)
def test_long_product(device, rows, n, k):
    _, codes, scale, w, there, want, off = operands(device, rows, n, k)
    y = fl.fp8_matmul(codes, scale, w)
    assert torch.equal(fl.fp8_matmul(codes, scale, w), y)
    got = codes_of(y[there])
    close(got, want, 2.0 ** -8 * np.abs(want) + off)
    assert np.linalg.norm(got - want) <= 2.0 ** -8 * np.linalg.norm(want)


@pytest.mark.parametrize("squares", [product_relu2, relu2_fast])
@pytest.mark.parametrize("rows,n,k", LONG + SIZES[-5:])
def test_long_product_relu2(device, rows, n, k, squares):
    _, codes, scale, w, there, h, off = operands(device, rows, n, k)
    a8, a_s = squares(codes, scale, w)
    want = np.maximum(h, 0.0) ** 2
    slack = 2 * np.maximum(h, 0.0) * off + off * off + 4 * EPS * want
    s = held(a_s[there])
    got = fb.values(codes_of(a8[there].contiguous()), exps_of(a_s[there]), 1)
    close(got, want, slack + np.maximum(2.0 ** -4 * (want + slack), 2.0 ** -10 * np.repeat(s, 128, 1)[:, :n]))
    pad = lambda t: np.pad(t, ((0, 0), (0, -n % 128))).reshape(len(h), -1, 128).max(-1)   # noqa: E731
    most, worst = pad(want), pad(slack)
    assert bool((most - worst <= 448 * s).all()) and bool(((most + worst > 224 * s) | (most == 0)).all())


@pytest.mark.parametrize("rows,n,k", LONG)
def test_long_product_relu2_backward(device, rows, n, k):
    gen, codes, scale, w, there, h, off = operands(device, rows, n, k)
    a8, a_s = fl.quantize_rows((uneven(gen, device, rows, n, 1).clamp(min=0) ** 2).to(device))
    root = 2 * np.sqrt(fb.values(codes_of(a8[there].contiguous()), exps_of(a_s[there]), 1))
    dh, q, q_s = product_relu2_bwd(codes, scale, w, a8, a_s)
    want = h * root
    got = codes_of(dh[there])
    close(got, want, 2.0 ** -8 * np.abs(want) + off * root + 4 * EPS * np.abs(want))
    some = there[::7]
    assert same_form(q[some], q_s[some], codes_of(dh[some]), 1)


@pytest.mark.parametrize("rows,n,k", [(33, 272, 144), (600, 4112, 128), (3000, 4112, 128)])
@pytest.mark.parametrize("least,most", [(1, 8), (8, 24), (120, 134), (232, 247)])
def test_square_roots_at_the_ends_of_the_range(device, rows, n, k, least, most):
    """Squared activations from fp32's smallest numbers, and below, to its largest: twice their roots lie far inside its range.
    Small, half and full tiles."""
    gen = torch.Generator().manual_seed(rows + least)
    codes, scale, x = form(gen, device, rows, k)
    w, wv = weight(gen, device, n, k)
    blocks = -(-n // 128)
    a8 = torch.randint(0, 0x78, (rows, n), generator=gen, dtype=torch.uint8).to(device).view(fl.CODES)   # 0 to 240
    e = torch.randint(least, most + 1, (rows, -(-blocks // 4) * 4), generator=gen, dtype=torch.uint8)
    e[torch.rand(e.shape, generator=gen) < 0.3] = 127   # beside ordinary ones
    a_s = e.to(device).view(fl.SCALE)[:, :blocks]
    root = 2 * np.sqrt(fb.values(codes_of(a8), exps_of(a_s), 1))
    dh, q, q_s = product_relu2_bwd(codes, scale, w, a8, a_s)
    want, off = (x @ wv.T) * root, (2.0 ** -10 + k * EPS) * (np.abs(x) @ np.abs(wv).T) * root
    close(codes_of(dh), want, 2.0 ** -8 * np.abs(want) + off + 4 * EPS * np.abs(want))
    assert same_form(q[:40], q_s[:40], codes_of(dh[:40]), 1)


def test_what_is_kept_may_wait_in_host_memory(device):
    """Saved tensors that go to the host and come back, weights held by the caller among them."""
    gen = torch.Generator().manual_seed(21)
    x, dy = bf(gen, 70, 256).to(device).requires_grad_(), bf(gen, 70, 144).to(device)
    w, fc, proj = ((torch.randn(*s, generator=gen) / 16).to(device).requires_grad_() for s in ((144, 256), (640, 256), (144, 640)))
    held_w, held_fc, held_proj = (fl.quantize_weight(t.detach(), True) for t in (w, fc, proj))

    def step():
        y = fl.checkpointed_linear(x, w, held_w) + fl.checkpointed_mlp(x, fc, proj, held_fc, held_proj)
        return y, (x, w, fc, proj)

    want = torch.autograd.grad(*step(), dy)
    with torch.autograd.graph.save_on_cpu():
        out = step()
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(*out, dy)))


# --- how exact the squares are

def dropped(x, w):
    """What the matrix cores may drop of x w^T: of each eight adjacent products seven times 2^-13 of the largest."""
    rows, k = x.shape
    x, w = np.abs(x).reshape(rows, 1, k // 8, 8), np.abs(w).reshape(1, -1, k // 8, 8)
    return 7 * 2.0 ** -13 * np.stack([(x[i] * w[0]).max(-1).sum(-1) for i in range(rows)])


def between(got, scale, h, off):
    """Whether 8-bit squares are those of sums within off of h, each rounded once: code for code, and the scales."""
    n = h.shape[1]
    lo, hi = np.maximum(h - off, 0.0) ** 2 * (1 - EPS), np.maximum(h + off, 0.0) ** 2 * (1 + EPS)
    top = lambda t: np.pad(t, ((0, 0), (0, -n % 128))).reshape(len(h), -1, 128).max(-1)   # noqa: E731
    least, most = fb.exponents(top(lo)), fb.exponents(top(hi))
    assert bool(((exps_of(scale) >= least) & (exps_of(scale) <= most)).all())
    s = np.repeat(held(scale), 128, 1)[:, :n]
    codes = codes_of(got.contiguous())
    low, high = fb.e4m3_round(np.minimum(lo / s, 448)), fb.e4m3_round(np.minimum(hi / s, 448))
    assert bool(((codes >= low) & (codes <= high)).all())


def others(codes, scale, h):
    """The share of 8-bit squares that are not float64's."""
    return (fb.values(codes_of(codes.contiguous()), exps_of(scale), 1) != fb.through(np.maximum(h, 0.0) ** 2, 1)).mean()


# few rows, small, half and full tiles, several tiles a workgroup
SQUARES = [(40, 272, 400), (65, 1280, 1168), (600, 4112, 1168), (3000, 4112, 128), (9300, 2064, 1168), (8190, 4352, 768)]


@pytest.mark.parametrize("rows,n,k", SQUARES)
def test_squares_of_exact_products(device, rows, n, k):
    """fp32 sums of exact products: a code may be another than float64's where the square lies that near to the border of two.
    How many do: a square is off by twice its sum's relative error d, codes lie 2^-4 to 2^-3 of a value apart, 0.09 in the mean: a
    share of 2 d / 0.09. k / 8 roundings of 2^-24 / sqrt(3), all of a result's own size, make d 4e-7 at k = 1,168: 1e-5; a tenfold of it
    is allowed, where the products by eights with their d of 1e-5 to 3e-5 give 2e-4 to 7e-4."""
    _, codes, scale, w, there, h, _ = operands(device, rows, n, k)
    x, wv = fb.values(codes_of(codes[there].contiguous()), exps_of(scale[there]), 1), fb.values(codes_of(w.codes), exps_of(w.scale), 128)
    a8, a_s = product_relu2(codes, scale, w)
    between(a8[there], a_s[there], h, k * EPS * (np.abs(x) @ np.abs(wv).T))
    assert others(a8[there], a_s[there], h) <= 1e-4
    again = product_relu2(codes, scale, w)
    assert torch.equal(again[0].view(torch.uint8), a8.view(torch.uint8))


@pytest.mark.parametrize("rows,n,k", SQUARES)
def test_squares_of_products_by_eights(device, rows, n, k):
    """The fast form's products drop bits in the larger tiles, by eights of columns, and no more than that."""
    _, codes, scale, w, there, h, _ = operands(device, rows, n, k)
    some = np.arange(0, len(h), max(1, len(h) // 24))
    there, h = there[torch.from_numpy(some).to(device)], h[some]
    x, wv = fb.values(codes_of(codes[there].contiguous()), exps_of(scale[there]), 1), fb.values(codes_of(w.codes), exps_of(w.scale), 128)
    a8, a_s = relu2_fast(codes, scale, w)
    between(a8[there], a_s[there], h, dropped(x, wv) + k * EPS * (np.abs(x) @ np.abs(wv).T))
    assert others(a8[there], a_s[there], h) <= 1e-3


@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("rows", [1, 40, 700, 9000])
def test_mlp_is_as_exact_as_its_squares(device, rows, fast):
    """An MLP's result is off by its own rounding alone, in any batch, but for the squares that the fast form takes otherwise; in
    training, too, whose gradients are of those squares."""
    gen = torch.Generator().manual_seed(rows)
    x = bf(gen, rows, 400).to(device)
    fc_w, proj_w = (torch.randn(*s, generator=gen).to(device) * s[1] ** -0.5 for s in ((2064, 400), (144, 2064)))
    fc, proj = fl.quantize_weight(fc_w, True), fl.quantize_weight(proj_w, True)
    z = fl.fp8_mlp(x, fc, proj, fast=fast)
    if not fast:
        fcv, pv = (fb.values(codes_of(t.codes), exps_of(t.scale), 128) for t in (fc, proj))
        at = torch.arange(0, rows, max(1, rows // 200))
        want = fb.through(np.maximum(fb.through(x[at].double().cpu().numpy(), 1) @ fcv.T, 0.0) ** 2, 1) @ pv.T
        assert np.linalg.norm(codes_of(z[at]) - want) <= 2.0 ** -8 * np.linalg.norm(want)
        assert torch.equal(fl.fp8_mlp(x, fc, proj), z)
    given = [t.clone().requires_grad_() for t in (x, fc_w, proj_w)]
    y = fl.checkpointed_mlp(*given, fast=fast)
    codes, scale = fl.quantize_rows(x)
    act = (relu2_fast if fast else product_relu2)(codes, scale, fc)
    assert torch.equal(y, fl.fp8_matmul(*act, proj)) and (rows <= 16 or torch.equal(y, z))
    dy = bf(gen, rows, 144).to(device)
    dx, dfc, dproj = torch.autograd.grad(y, given, dy)
    dh, q, q_s = product_relu2_bwd(*fl.quantize_rows(dy), fl.Fp8Weight(proj.codes_t, proj.scale_t), *act)
    assert torch.equal(dx, fl.fp8_matmul(q, q_s, fl.Fp8Weight(fc.codes_t, fc.scale_t)))
    for got, left, right in ((dfc, dh, (codes, scale)), (dproj, dy, act)):
        a, b = left.double().cpu().numpy(), fb.values(codes_of(right[0]), exps_of(right[1]), 1)
        close(codes_of(got), a.T @ b, (rows + 300) * EPS * (np.abs(a).T @ np.abs(b)))


# --- gradients against differences, where nothing is rounded

def whole_numbers(gen, rows, cols, of):
    """0, +-1, +-2 and +-3."""
    return torch.randint(-3, 4, (rows, cols), generator=gen).float()


def one_a_row(gen, rows, cols):
    """One number of 1 and 2 in each row, of either sign, anywhere."""
    t = torch.zeros(rows, cols)
    t[torch.arange(rows), torch.randint(0, cols, (rows,), generator=gen)] = (
        torch.randint(1, 3, (rows,), generator=gen) * (2 * torch.randint(0, 2, (rows,), generator=gen) - 1)).float()
    return t


def directions(gen, shape):
    """Single entries, then one row, one column, and a few entries over all of it."""
    rows, cols = shape
    entries = [(int(torch.randint(0, rows, (1,), generator=gen)), int(torch.randint(0, cols, (1,), generator=gen)))
               for _ in range(12)] + [(0, 0), (rows - 1, cols - 1)]
    for i, j in entries:
        v = torch.zeros(shape, dtype=torch.float64)
        v[i, j] = 1.0
        yield v
    for at in (np.s_[rows // 2, :], np.s_[:, cols // 3]):
        v = torch.zeros(shape, dtype=torch.float64)
        v[at] = 1.0
        yield v
    yield (torch.rand(shape, generator=gen) < 0.02).double()


STEP = 2.0 ** -20


def compare(gen, loss, inputs, grads, kink):
    """<gradient, v> against (L(+v) - L(-v)) / 2 in float64 for directions of few entries. L is a square of what relu lets through at
    most, so the difference is the derivative but at relu's border, where it adds at most STEP / 2 kink for an entry of v, and for
    float64's own rounding of L. Half and twice the gradient have to fail where there is one."""
    told = 0
    for i, g in enumerate(grads):
        g = g.detach().double().cpu()
        slack = 2.0 ** -8 if inputs[i].dtype == torch.bfloat16 else EPS
        at = [t.double() for t in inputs]
        for v in directions(gen, tuple(g.shape)):
            plus, minus = (loss(*(t + s * STEP * v if j == i else t for j, t in enumerate(at))) for s in (1, -1))
            want, size = (plus - minus) / (2 * STEP), float((g.abs() * v).sum())
            off = size * slack + float(v.sum()) ** 2 * kink * STEP / 2 + 2.0 ** -50 * (abs(plus) + abs(minus) + 1) / STEP
            got = float((g * v).sum())
            assert abs(got - want) <= off, (i, got, want, off)
            if abs(want) > 8 * off:
                told += 1
                assert abs(got / 2 - want) > off and abs(2 * got - want) > off
    assert told >= 6 * len(grads)


@pytest.mark.parametrize("m,c,f,n", [(500, 144, 384, 80), (700, 272, 1040, 160)])
def test_gradients_of_whole_numbers_by_differences(device, m, c, f, n):
    """Inputs whose 8-bit forms, sums, squares and gradients before the square are all exact: x and dy have one number a row, so a
    sum before the square is one of 0, 1, 2, 3, 4 and 6, its square has four bits at most, as has dh = da 2 sqrt(a) (1, 3 or 9
    times a power of two). What is left is dx's rounding to bf16."""
    gen = torch.Generator().manual_seed(30)
    x, dy = one_a_row(gen, m, c).to(torch.bfloat16), one_a_row(gen, m, n).to(torch.bfloat16)
    fc, proj, w = whole_numbers(gen, f, c, 128), whole_numbers(gen, n, f, 128), whole_numbers(gen, n, c, 128)
    asked = lambda *ts: [t.to(device).requires_grad_() for t in ts]   # noqa: E731
    given = asked(x, fc, proj)
    got = torch.autograd.grad(fl.checkpointed_mlp(*given), given, dy.to(device))

    def mlp(x, fc, proj):
        return float(((x @ fc.t()).clamp(min=0).square() @ proj.t() * dy.double()).sum())

    # an entry's border: at most 3 rows (of fc) or numbers (of x) squared times a da of 6, for each row or output that it reaches
    compare(gen, mlp, (x, fc, proj), got, 9 * 6 * max(m, f))
    given = asked(x, w)
    got = torch.autograd.grad(fl.checkpointed_linear(*given), given, dy.to(device))
    compare(gen, lambda x, w: float(((x @ w.t()) * dy.double()).sum()), (x, w), got, 0)
