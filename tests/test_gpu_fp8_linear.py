"""The 8-bit linear layers on the GPU against float64 on the CPU (oracle/fp8_block.py): the 8-bit form bit for bit; products,
the ReLU^2 form and its gradient, and weight gradients from checkpoints, at sizes around blocks, tiles and slices; the training
ops' gradients by formula and by differences; strides, NaN, streams, captured steps, and what is kept for the backward.

Bounds. A product of two e4m3 values is exact. Of eight products of adjacent k the matrix cores keep bits down to 2^-13 of the
largest, so each of the other seven loses less than 2^-13 of it: at most 7 2^-13 < 2^-10 of the eight's sum of magnitudes. The
rest is fp32: a sum of n terms in any order is within n 2^-23 of the sum of magnitudes. A bf16 result adds half a step,
2^-8 of the value at most, an 8-bit one 2^-4 of the value or 2^-10 of its block's scale."""
import numpy as np
import pytest
import torch

from nanochat_amd import fp8_linear as fl, native
from nanochat_amd.native import hip_library, stream
from oracle import fp8_block as fb

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -23
BF16, F32 = torch.bfloat16, torch.float32


def bf(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(BF16)


def rowwise(gen, rows, cols):
    """bf16 rows of sizes over several powers of two, a few channels far above the others."""
    x = torch.randn(rows, cols, generator=gen) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=gen).float())
    return (x * torch.where(torch.rand(cols, generator=gen) < 0.02, 16.0, 1.0)).to(BF16)


def codes_of(t):
    return t.cpu().float().double().numpy()


def exps_of(t):
    return t.cpu().view(torch.uint8).numpy().astype(np.int64) - 127 if t.is_contiguous() else exps_of(t.contiguous())


def same_form(codes, scale, x, rows):
    want, exps = fb.quantize(x, rows)
    return np.array_equal(codes_of(codes), want, equal_nan=True) and np.array_equal(exps_of(scale), exps)


def held(scale):
    """The same scales, of a device tensor, as plain numbers."""
    return np.ldexp(1.0, exps_of(scale))


def form(gen, device, rows, cols, spread=True):
    """Activations in the 8-bit form on the device, and their values."""
    codes, scale = fl.quantize_rows((rowwise(gen, rows, cols) if spread else bf(gen, rows, cols)).to(device))
    return codes, scale, fb.values(codes_of(codes), exps_of(scale), 1)


def weight(gen, device, n, k, transpose=False):
    w = fl.quantize_weight((torch.randn(n, k, generator=gen) * k ** -0.5).to(device), transpose)
    return w, fb.values(codes_of(w.codes), exps_of(w.scale), 128)


def product_relu2(codes, scale, w):
    rows, k = codes.shape
    n = w.codes.size(0)
    out, out_scale = torch.empty(rows, n, dtype=fl.CODES, device=codes.device), fl._new_scale(codes, rows, n)
    native.check(hip_library().nc_fp8_matmul_relu2(codes.data_ptr(), scale.data_ptr(), scale.stride(0), w.codes.data_ptr(),
                                                   w.scale.data_ptr(), w.scale.stride(0), rows, n, k, out.data_ptr(),
                                                   out_scale.data_ptr(), out_scale.stride(0), stream()))
    return out, out_scale


def product_relu2_bwd(codes, scale, w, act, act_scale):
    rows, k = codes.shape
    n = w.codes.size(0)
    out, q = torch.empty(rows, n, dtype=BF16, device=codes.device), torch.empty_like(act)
    q_scale = fl._new_scale(codes, rows, n)
    native.check(hip_library().nc_fp8_matmul_relu2_bwd(
        codes.data_ptr(), scale.data_ptr(), scale.stride(0), w.codes.data_ptr(), w.scale.data_ptr(), w.scale.stride(0), rows, n, k,
        act.data_ptr(), act_scale.data_ptr(), act_scale.stride(0), out.data_ptr(), q.data_ptr(), q_scale.data_ptr(),
        q_scale.stride(0), stream()))
    return out, q, q_scale


# --- the 8-bit form

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 128), (3, 144), (33, 400), (129, 1664), (7, 5008)])
def test_rows(device, rows, cols, dtype):
    gen = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=gen) * torch.exp2(torch.randint(-40, 40, (rows, cols), generator=gen).float())
    x[0] = 0.0
    x = x.to(dtype)
    codes, scale = fl.quantize_rows(x.to(device))
    assert same_form(codes, scale, x.double().numpy(), 1)
    assert fl.quantize_rows(x.to(device)[:0])[0].shape == (0, cols)


def test_rows_at_the_ends_of_the_range(device):
    """The largest and smallest numbers of each type, powers of two and 1.75 times them, and one value in each block's way."""
    for dtype in (BF16, F32):
        top = torch.finfo(dtype).max
        ends = [top, -top, torch.finfo(dtype).tiny, 2.0 ** -133, 448.0, 449.0 if dtype == F32 else 450.0, 1.75, 1.7578125, 0.0]
        x = torch.zeros(len(ends) * 2, 256)
        for i, v in enumerate(ends):
            x[2 * i, 17], x[2 * i + 1, 255], x[2 * i + 1, 128] = v, v, v / 3
        x = x.to(dtype)
        codes, scale = fl.quantize_rows(x.to(device))
        assert same_form(codes, scale, x.double().numpy(), 1), dtype


def test_rows_of_any_stride_and_alignment(device):
    gen = torch.Generator().manual_seed(1)
    wide = rowwise(gen, 20, 1000).to(device)
    for x in (wide[:, 8:408], wide[:, 3:403], wide[::3, 16:272], wide.t()[:400, :16], wide[:5].expand(5, 1000)[:, :144],
              wide[0].expand(4, 1000)[:, :160], wide[:, :960].view(4, 5, 960), wide[2, :144]):
        for y in (x, x.float() if x.stride(-1) != 1 else torch.as_strided(wide.float(), x.shape, x.stride(), x.storage_offset())):
            codes, scale = fl.quantize_rows(y)
            assert same_form(codes, scale, y.double().reshape(-1, y.size(-1)).cpu().numpy(), 1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_blocks_that_are_not_finite(device, bad):
    """A block with such a value is NaN, and so is what is made from it; its neighbours keep theirs."""
    gen = torch.Generator().manual_seed(2)
    for dtype in (BF16, F32):
        x = rowwise(gen, 40, 384).to(dtype)
        x[5, 200] = bad
        codes, scale = fl.quantize_rows(x.to(device))
        assert same_form(codes, scale, x.double().numpy(), 1)
        w, wv = weight(gen, device, 144, 384)
        y = fl.fp8_matmul(codes, scale, w)
        assert bool(torch.isnan(y[5]).all()) and not bool(torch.isnan(y[[4, 6]]).any())
        a8, a_s = product_relu2(codes, scale, w)
        assert bool(torch.isnan(a8[5].float()).all()) and not bool(torch.isnan(a8[[4, 6]].float()).any())
        dy = bf(gen, 40, 144).to(device)
        dw = fl.checkpoint_weight_grad(dy, codes, scale)
        assert torch.isnan(dw).any(0).tolist() == [128 <= k < 256 for k in range(384)]
    v = torch.randn(300, 272, generator=gen)
    v[140, 30] = bad
    q = fl.quantize_weight(v.to(device)[:288], True)
    assert same_form(q.codes, q.scale, v[:288].double().numpy(), 128)
    assert torch.equal(q.codes_t.view(torch.uint8), q.codes.view(torch.uint8).t())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(16, 16), (128, 128), (144, 400), (640, 272), (1, 128), (300, 144)])
def test_weights(device, n, k, dtype):
    gen = torch.Generator().manual_seed(n + k)
    w = (torch.randn(n, k, generator=gen) * torch.exp2(torch.randint(-20, 20, (n, k), generator=gen).float())).to(dtype)
    for transpose in (False, True) if n % 16 == 0 else (False,):
        for t in (w.to(device), torch.cat([w, w], 1).to(device)[:, 16 * (k // 32):][:, :k]):
            q = fl.quantize_weight(t, transpose)
            assert same_form(q.codes, q.scale, t.double().cpu().numpy(), 128)
            if transpose:
                assert torch.equal(q.codes_t.view(torch.uint8), q.codes.view(torch.uint8).t())
                assert np.array_equal(exps_of(q.scale_t), exps_of(q.scale).T)


# --- products

SIZES = [(1, 16, 16), (1, 128, 128), (2, 272, 144), (17, 128, 640), (63, 400, 512), (64, 144, 2000), (65, 1280, 128),
         (130, 256, 400), (257, 528, 272), (600, 4112, 128), (3000, 1680, 400), (4100, 4112, 144), (9000, 2064, 272)]


def close(got, want, slack):
    off = np.abs(got - want)
    assert np.isfinite(got).all() and bool((off <= slack).all()), float((off / np.maximum(slack, 1e-300)).max())


@pytest.mark.parametrize("rows,n,k", SIZES)
def test_product(device, rows, n, k):
    gen = torch.Generator().manual_seed(rows + n + k)
    codes, scale, x = form(gen, device, rows, k)
    w, wv = weight(gen, device, n, k)
    y = fl.fp8_matmul(codes, scale, w)
    again = fl.fp8_matmul(codes, scale, w)
    assert torch.equal(y, again)
    want, mag = x @ wv.T, np.abs(x) @ np.abs(wv).T
    close(codes_of(y), want, 2.0 ** -8 * np.abs(want) + (2.0 ** -10 + k * EPS) * mag)
    # far closer as a rule: a wrong block's scale or a lost row would show here
    assert np.linalg.norm(codes_of(y) - want) <= 2.0 ** -8 * np.linalg.norm(want)


@pytest.mark.parametrize("rows,n,k", SIZES)
def test_product_relu2(device, rows, n, k):
    gen = torch.Generator().manual_seed(rows + n + k)
    codes, scale, x = form(gen, device, rows, k)
    w, wv = weight(gen, device, n, k)
    a8, a_s = product_relu2(codes, scale, w)
    h, off = x @ wv.T, (2.0 ** -10 + k * EPS) * (np.abs(x) @ np.abs(wv).T)
    want = np.maximum(h, 0.0) ** 2
    slack = 2 * np.maximum(h, 0.0) * off + off * off + 4 * EPS * want
    got = fb.values(codes_of(a8), exps_of(a_s), 1)
    s = np.repeat(held(a_s), 128, 1)[:, :n]
    close(got, want, slack + np.maximum(2.0 ** -4 * (want + slack), 2.0 ** -10 * s))
    # the scale is the least that holds its block, of the kernel's own sums
    pad = lambda t: np.pad(t, ((0, 0), (0, -n % 128))).reshape(rows, -1, 128).max(-1)   # noqa: E731
    most, worst = pad(want), pad(slack)
    assert bool((most - worst <= 448 * held(a_s)).all())
    assert bool(((most + worst > 224 * held(a_s)) | (most == 0)).all())


@pytest.mark.parametrize("rows,n,k", SIZES)
def test_product_relu2_backward(device, rows, n, k):
    gen = torch.Generator().manual_seed(rows + n + k)
    codes, scale, x = form(gen, device, rows, k)
    w, wv = weight(gen, device, n, k)
    a8, a_s = fl.quantize_rows((rowwise(gen, rows, n).float().clamp(min=0) ** 2).to(device))
    root = 2 * np.sqrt(fb.values(codes_of(a8), exps_of(a_s), 1))
    dh, q, q_s = product_relu2_bwd(codes, scale, w, a8, a_s)
    want, off = (x @ wv.T) * root, (2.0 ** -10 + k * EPS) * (np.abs(x) @ np.abs(wv).T) * root
    close(codes_of(dh), want, 2.0 ** -8 * np.abs(want) + off + 4 * EPS * np.abs(want))
    assert same_form(q, q_s, codes_of(dh), 1)


@pytest.mark.parametrize("rows,n,k", [(65, 1280, 128), (600, 4112, 128), (3000, 4112, 128), (9000, 2064, 272)])
def test_products_write_their_results_and_nothing_else(device, rows, n, k):
    """Results of small, half, full and both tiles in the middle of larger buffers: 300 rows before and behind them, and the scales'
    other columns, stay."""
    gen = torch.Generator().manual_seed(rows)
    codes, scale, _ = form(gen, device, rows, k)
    w, _ = weight(gen, device, n, k)
    a8, a_s = product_relu2(codes, scale, w)
    dh, q, q_s = product_relu2_bwd(codes, scale, w, a8, a_s)
    y, blocks, pitch, guard = fl.fp8_matmul(codes, scale, w), a_s.size(1), 4 * ((n + 127) // 128 // 4 + 2), 300

    def around(width):
        whole = torch.full((rows + 2 * guard, width), 0xA5, dtype=torch.uint8, device=device)
        return whole, whole[guard:].data_ptr()

    def check(whole, want):
        inside = whole[guard:guard + rows, :want.size(1)]
        assert torch.equal(inside, want)
        inside.fill_(0xA5)
        assert bool((whole == 0xA5).all())

    head = (codes.data_ptr(), scale.data_ptr(), scale.stride(0), w.codes.data_ptr(), w.scale.data_ptr(), w.scale.stride(0), rows, n, k)
    raw = lambda v: v.contiguous().view(torch.uint8)   # noqa: E731
    lib = hip_library()
    out, out_at = around(2 * n)
    native.check(lib.nc_fp8_matmul(*head, out_at, stream()))
    check(out, raw(y))
    form_, form_at = around(n)
    exps, exps_at = around(pitch)
    native.check(lib.nc_fp8_matmul_relu2(*head, form_at, exps_at, pitch, stream()))
    check(form_, raw(a8))
    check(exps, raw(a_s)[:, :blocks])
    native.check(lib.nc_fp8_matmul_relu2_bwd(*head, a8.data_ptr(), a_s.data_ptr(), a_s.stride(0), out_at, form_at, exps_at, pitch,
                                             stream()))
    check(out, raw(dh))
    check(form_, raw(q))
    check(exps, raw(q_s)[:, :blocks])


def test_product_of_everyone_elses_scales(device):
    """Scales of other tensors than quantize_rows makes: a wider pitch, and exponents far apart in one row."""
    gen = torch.Generator().manual_seed(3)
    codes, _, _ = form(gen, device, 70, 1200)
    e = torch.randint(100, 150, (70, 40), generator=gen, dtype=torch.uint8).to(device)
    scale = e.view(torch.float8_e8m0fnu)[:, 8:18]
    w, wv = weight(gen, device, 144, 1200)
    x = fb.values(codes_of(codes), exps_of(scale), 1)
    want, mag = x @ wv.T, np.abs(x) @ np.abs(wv).T
    close(codes_of(fl.fp8_matmul(codes, scale, w)), want, 2.0 ** -8 * np.abs(want) + (2.0 ** -10 + 1200 * EPS) * mag)


@pytest.mark.parametrize("rows", [0, 1, 5, 16, 17, 40, 128, 129, 700])
def test_serving_layers(device, rows):
    """fp8_linear and fp8_mlp give what their parts give, from any leading dimensions and strides."""
    gen = torch.Generator().manual_seed(rows)
    x = rowwise(gen, rows, 640).to(device)
    w, wv = weight(gen, device, 272, 640)
    x8 = fb.through(x.double().cpu().numpy(), 1) if rows else np.zeros((0, 640))
    want, mag = x8 @ wv.T, np.abs(x8) @ np.abs(wv).T
    y = fl.fp8_linear(x, w)
    assert y.shape == (rows, 272)
    close(codes_of(y), want, 2.0 ** -8 * np.abs(want) + (2.0 ** -10 + 640 * EPS) * mag)
    wide = torch.zeros(rows, 1000, dtype=BF16, device=device)
    wide[:, 8:648] = x
    assert torch.equal(fl.fp8_linear(wide[:, 8:648], w), y)
    assert torch.equal(fl.fp8_linear(x.view(rows, 1, 640), w), y.view(rows, 1, 272))
    fc, fcv = weight(gen, device, 1040, 640)
    proj, pv = weight(gen, device, 160, 1040)
    z = fl.fp8_mlp(x, fc, proj)
    assert z.shape == (rows, 160) and torch.equal(fl.fp8_mlp(wide[:, 8:648], fc, proj), z)
    if not rows:
        return
    h, off = x8 @ fcv.T, (2.0 ** -10 + 640 * EPS) * (np.abs(x8) @ np.abs(fcv).T)
    a = np.maximum(h, 0.0) ** 2
    # each squared activation is off by its sum's error, one rounding to 8 bits, and half the smallest step of its block
    top = np.pad(a, ((0, 0), (0, -1040 % 128))).reshape(rows, -1, 128).max(-1)
    err = 2 * np.maximum(h, 0.0) * off + off * off
    err = err + 2.0 ** -4 * (a + err) + 2.0 ** -10 * np.repeat(top / 128, 128, 1)[:, :1040]
    close(codes_of(z), a @ pv.T, err @ np.abs(pv).T + 2.0 ** -8 * np.abs(a @ pv.T) + (2.0 ** -10 + 1040 * EPS) * ((a + err) @ np.abs(pv).T))
    exact = fb.through(a, 1) @ pv.T
    assert np.linalg.norm(codes_of(z) - exact) <= 2.0 ** -6 * np.linalg.norm(exact)


# by the number of rows, of outputs, and of (16 outputs) x (32 rows) against the CUs (256)
FEW = [(rows, 400, 2064) for rows in (1, 2, 8, 9, 15, 16, 17, 31, 32, 33, 100, 127, 128)]
FEW += [(1, 16, 20000), (16, 33024, 144), (3, 4992, 400), (20, 48, 16400), (20, 4800, 272), (32, 33024, 144), (40, 4816, 144),
        (64, 2064, 1296), (97, 9616, 144), (128, 33040, 272), (128, 16, 16384), (77, 16, 16),
        (37, 1280, 1280), (49, 4096, 16), (64, 144, 1280), (64, 784, 400)]


@pytest.mark.parametrize("rows,n,k", FEW)
def test_few_rows(device, rows, n, k):
    """Up to 128 rows, which read the weight once: from rows of any alignment, from codes, and with nothing written behind them."""
    gen = torch.Generator().manual_seed(rows + n + k)
    x = rowwise(gen, rows, k)
    w, wv = weight(gen, device, n, k)
    x8 = fb.through(x.double().numpy(), 1)
    want, mag = x8 @ wv.T, np.abs(x8) @ np.abs(wv).T
    slack = 2.0 ** -8 * np.abs(want) + (2.0 ** -10 + k * EPS) * mag
    odd = torch.zeros(rows, k + 3, dtype=BF16, device=device)
    odd[:, 1:k + 1] = x.to(device)
    padded = torch.full((rows, k + 24), float("nan"), dtype=BF16, device=device)
    padded[:, 16:k + 16] = x.to(device)
    for y in (fl.fp8_linear(x.to(device), w), fl.fp8_linear(odd[:, 1:k + 1], w), fl.fp8_linear(padded[:, 16:k + 16], w),
              fl.fp8_matmul(*fl.quantize_rows(x.to(device)), w)):
        close(codes_of(y), want, slack)
        assert np.linalg.norm(codes_of(y) - want) <= 2.0 ** -8 * np.linalg.norm(want)
    lib, out = hip_library(), torch.full((rows + 1, n), 7.0, dtype=BF16, device=device)
    xd, xf = x.to(device), x.float().to(device)
    for t, f32 in ((xd, 0), (xf, 1)):
        need = lib.nc_fp8_linear_workspace_bytes(t.data_ptr(), f32, k, rows, n, k)
        ws = torch.full((need + 64,), 9, dtype=torch.uint8, device=device)
        assert lib.nc_fp8_linear(t.data_ptr(), f32, k, w.codes.data_ptr(), w.scale.data_ptr(), w.scale.stride(0), rows, n, k,
                                 out.data_ptr(), ws.data_ptr(), need, stream()) == 0
        close(codes_of(out[:rows]), want, slack)
        assert bool((out[rows] == 7).all()) and bool((ws[need:] == 9).all())


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 33, 128])
@pytest.mark.parametrize("c,hidden,n", [(400, 2064, 144), (144, 9616, 32), (1280, 528, 4816)])
def test_few_rows_mlp(device, rows, c, hidden, n):
    """An MLP's squared activations from exact products: their codes are those of float64's, but for values that lie on the border
    of two codes, and the result is off by its own rounding alone."""
    gen = torch.Generator().manual_seed(rows + c + n)
    x = rowwise(gen, rows, c)
    fc, fcv = weight(gen, device, hidden, c)
    proj, pv = weight(gen, device, n, hidden)
    want = fb.through(np.maximum(fb.through(x.double().numpy(), 1) @ fcv.T, 0.0) ** 2, 1) @ pv.T
    lib, out = hip_library(), torch.full((rows + 1, n), 7.0, dtype=BF16, device=device)
    need = lib.nc_fp8_mlp_workspace_bytes(rows, c, hidden)
    ws, xd = torch.full((need + 64,), 9, dtype=torch.uint8, device=device), x.to(device)
    assert lib.nc_fp8_mlp(xd.data_ptr(), c, fc.codes.data_ptr(), fc.scale.data_ptr(), fc.scale.stride(0), proj.codes.data_ptr(),
                          proj.scale.data_ptr(), proj.scale.stride(0), rows, c, hidden, n, out.data_ptr(), ws.data_ptr(), need,
                          stream()) == 0
    assert bool((out[rows] == 7).all()) and bool((ws[need:] == 9).all())
    z = fl.fp8_mlp(xd, fc, proj)
    assert torch.equal(z, out[:rows])
    assert np.linalg.norm(codes_of(z) - want) <= 2.0 ** -8 * np.linalg.norm(want)


@pytest.mark.parametrize("rows", [5, 12, 40, 140])
def test_rows_that_are_not_finite(device, rows):
    """A NaN or an infinity makes its own row NaN and no other."""
    gen = torch.Generator().manual_seed(rows)
    x = rowwise(gen, rows, 400).to(device)
    w, fc, proj = (weight(gen, device, *s)[0] for s in ((272, 400), (640, 400), (144, 640)))
    y, z = fl.fp8_linear(x, w), fl.fp8_mlp(x, fc, proj)
    bad = x.clone()
    bad[1, 7], bad[3, 300] = float("nan"), float("inf")
    ill = torch.zeros(rows, dtype=torch.bool, device=device)
    ill[1] = ill[3] = True
    for got, want in ((fl.fp8_linear(bad, w), y), (fl.fp8_mlp(bad, fc, proj), z)):
        assert bool(got[ill].isnan().all()) and torch.equal(got[~ill], want[~ill])


# --- weight gradients

@pytest.mark.parametrize("rows,n,k", [(1, 16, 16), (31, 8, 144), (33, 264, 128), (128, 272, 272), (300, 520, 2064),
                                      (2400, 640, 400), (9995, 1280, 1280), (4099, 16, 2048), (1500, 4104, 4112)])
def test_weight_gradient(device, rows, n, k):
    gen = torch.Generator().manual_seed(rows)
    codes, scale, x = form(gen, device, rows, k)
    dy = bf(gen, rows, n)
    a = dy.double().numpy()
    want, mag = a.T @ x, np.abs(a).T @ np.abs(x)
    got = fl.checkpoint_weight_grad(dy.to(device), codes, scale)
    slack = (rows + 300) * EPS * mag
    close(codes_of(got), want, slack)
    assert torch.equal(fl.checkpoint_weight_grad(dy.to(device), codes, scale), got)
    close(codes_of(fl.checkpoint_weight_grad(dy.to(device), codes, scale, dtype=BF16)), want, slack + 2.0 ** -8 * np.abs(want))
    start = torch.randn(n, k, generator=gen)
    buf = torch.full((n * k + 4096,), 7.0, device=device)
    out = buf[:n * k].view(n, k)
    out.copy_(start)
    assert fl.checkpoint_weight_grad(dy.to(device), codes, scale, out=out) is out
    s = start.double().numpy()
    close(codes_of(out), want + s, (rows + 300) * EPS * (mag + np.abs(s)))
    assert bool((buf[n * k:] == 7).all())


def test_weight_gradient_of_no_rows(device):
    codes, scale = fl.quantize_rows(torch.zeros(0, 128, dtype=BF16, device=device))
    dy, out = torch.zeros(0, 32, dtype=BF16, device=device), torch.ones(32, 128, device=device)
    assert not bool(fl.checkpoint_weight_grad(dy, codes, scale).any())
    assert bool((fl.checkpoint_weight_grad(dy, codes, scale, out=out) == 1).all())


# --- training

def formula_linear(x, w, dy):
    x8, w8 = fb.through(x, 1), fb.through(w, 128)
    dy8 = fb.through(dy, 1)
    return x8, w8, dy8, x8 @ w8.T, dy8 @ w8, dy.T @ x8


@pytest.mark.parametrize("shape,n,dtype,given,into", [((5, 7, 400), 272, F32, False, False), ((300, 128), 144, BF16, True, False),
                                                      ((2, 200, 256), 640, F32, True, True), ((1, 16), 16, BF16, False, True)])
def test_training_linear(device, shape, n, dtype, given, into):
    gen = torch.Generator().manual_seed(n)
    k = shape[-1]
    x = rowwise(gen, int(np.prod(shape[:-1])), k).view(shape).to(device).requires_grad_()
    w = (torch.randn(n, k, generator=gen) * k ** -0.5).to(dtype).to(device).requires_grad_()
    dy = bf(gen, *shape[:-1], n, scale=1e-3).to(device)
    buf = torch.ones(n, k, device=device) if into else None
    y = fl.checkpointed_linear(x, w, fl.quantize_weight(w.detach(), True) if given else None, buf)
    y.backward(dy)
    xd, wd, dyd = (t.detach().double().cpu().numpy().reshape(-1, t.size(-1)) for t in (x, w, dy))
    x8, w8, dy8, want_y, want_dx, want_dw = formula_linear(xd, wd, dyd)
    m = xd.shape[0]
    for got, want, mag, depth in ((y, want_y, np.abs(x8) @ np.abs(w8).T, k), (x.grad, want_dx, np.abs(dy8) @ np.abs(w8), n)):
        assert got.dtype == BF16
        close(codes_of(got.detach()).reshape(want.shape), want, 2.0 ** -8 * np.abs(want) + (2.0 ** -10 + depth * EPS) * mag)
    mag = np.abs(dyd).T @ np.abs(x8)
    if into:
        assert w.grad is None
        close(codes_of(buf), want_dw + 1, (m + 300) * EPS * (mag + 1))
    else:
        assert w.grad.dtype == dtype
        close(codes_of(w.grad), want_dw, (m + 300) * EPS * mag + (2.0 ** -8 * np.abs(want_dw) if dtype == BF16 else 0))


@pytest.mark.parametrize("m,c,f,n,dtype", [(1, 16, 32, 16, BF16), (130, 256, 1040, 256, BF16), (700, 144, 640, 272, F32)])
def test_training_mlp(device, m, c, f, n, dtype):
    """Against the formula, with the checkpoint of the squared activations as the kernel rounded it (that rounding is
    test_product_relu2's)."""
    gen = torch.Generator().manual_seed(m)
    x = rowwise(gen, m, c).to(device).requires_grad_()
    fc = (torch.randn(f, c, generator=gen) * c ** -0.5).to(dtype).to(device).requires_grad_()
    proj = (torch.randn(n, f, generator=gen) * f ** -0.5).to(dtype).to(device).requires_grad_()
    dy = bf(gen, m, n, scale=1e-3).to(device)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        y = fl.checkpointed_mlp(x, fc, proj)
    # what is kept: both 8-bit forms and the weights' transposes, nothing of x's or the sums' size in more than 8 bits
    assert sum(t.numel() * t.element_size() for t in kept) <= (m * (c + f) + f * (c + n)) * (1 + 1 / 8) + 4 * (2 * m + c + f)
    dx, dfc, dproj = torch.autograd.grad(y, (x, fc, proj), dy)
    xd, fd, pd, dyd = (t.detach().double().cpu().numpy() for t in (x, fc, proj, dy))
    x8, f8, p8, dy8 = fb.through(xd, 1), fb.through(fd, 128), fb.through(pd, 128), fb.through(dyd, 1)
    q = fl.quantize_weight(fc.detach())
    codes, scale = fl.quantize_rows(x.detach())
    a8, a_s = product_relu2(codes, scale, q)
    a = fb.values(codes_of(a8), exps_of(a_s), 1)
    close(codes_of(y.detach()), a @ p8.T, 2.0 ** -8 * np.abs(a @ p8.T) + (2.0 ** -10 + f * EPS) * (a @ np.abs(p8).T))
    mag = np.abs(dyd).T @ a
    close(codes_of(dproj), dyd.T @ a, (m + 300) * EPS * mag + (2.0 ** -8 * np.abs(dyd.T @ a) if dtype == BF16 else 0))
    dh, root = (dy8 @ p8) * 2 * np.sqrt(a), 2 * np.sqrt(a)
    off = (2.0 ** -10 + n * EPS) * (np.abs(dy8) @ np.abs(p8)) * root + 2.0 ** -8 * np.abs(dh) + 4 * EPS * np.abs(dh)
    want = dh.T @ x8
    close(codes_of(dfc), want, off.T @ np.abs(x8) + (m + 300) * EPS * ((np.abs(dh) + off).T @ np.abs(x8)) +
          (2.0 ** -8 * (np.abs(want) + off.T @ np.abs(x8)) if dtype == BF16 else 0))
    top = np.pad(np.abs(dh) + off, ((0, 0), (0, -f % 128))).reshape(m, -1, 128).max(-1)
    off8 = off + 2.0 ** -4 * (np.abs(dh) + off) + 2.0 ** -10 * np.repeat(top / 128, 128, 1)[:, :f]
    want, m8 = dh @ f8, (np.abs(dh) + off8) @ np.abs(f8)
    close(codes_of(dx), want, off8 @ np.abs(f8) + (2.0 ** -10 + f * EPS) * m8 + 2.0 ** -8 * m8)


@pytest.mark.parametrize("rows", [1, 33, 700, 9000])
@pytest.mark.parametrize("fc_type,proj_type,add", [(F32, F32, False), (BF16, BF16, False), (F32, BF16, False), (F32, F32, True)])
def test_both_weight_gradients_of_an_mlp(device, rows, fc_type, proj_type, add):
    """dfc and dproj, which may share a launch, against float64 from the operands that the op's own parts make."""
    gen = torch.Generator().manual_seed(rows)
    c, hidden, n = 272, 1040, 144
    x, dy = rowwise(gen, rows, c).to(device), bf(gen, rows, n).to(device)
    fc = (torch.randn(hidden, c, generator=gen) / 16).to(fc_type).to(device).requires_grad_()
    proj = (torch.randn(n, hidden, generator=gen) / 32).to(proj_type).to(device).requires_grad_()
    buffers = [torch.full(w.shape, 3.0, device=device) for w in (fc, proj)] if add else [None, None]
    y = fl.checkpointed_mlp(x, fc, proj, fc_grad=buffers[0], proj_grad=buffers[1])
    got = torch.autograd.grad(y, (fc, proj), dy, allow_unused=True) if not add else (y.backward(dy), buffers)[1]
    x8 = fl.quantize_rows(x)
    f8, p8 = fl.quantize_weight(fc.detach(), True), fl.quantize_weight(proj.detach(), True)
    act = product_relu2(*x8, f8)
    dh = product_relu2_bwd(*fl.quantize_rows(dy), fl.Fp8Weight(p8.codes_t, p8.scale_t), *act)[0]
    full = lambda codes, scale: torch.from_numpy(fb.values(codes_of(codes), exps_of(scale), 1))   # noqa: E731
    for g, left, right, t in zip(got, (dh, dy), (full(*x8), full(*act)), (fc_type, proj_type)):
        left = left.double().cpu()
        want, mag = left.t() @ right + (3.0 if add else 0.0), left.abs().t() @ right.abs() + (3.0 if add else 0.0)
        close(codes_of(g), want.numpy(), (mag * (rows + 2) * EPS + (2.0 ** -8 * want.abs() if t == BF16 else 0.0)).numpy())


def test_one_buffer_for_two_uses(device):
    """A weight used twice adds both its gradients to one buffer, which may be cleared between the forward and the backward."""
    gen = torch.Generator().manual_seed(11)
    w, x, dy = (torch.randn(256, 256, generator=gen) / 16).to(device), bf(gen, 70, 256).to(device), bf(gen, 70, 256).to(device)
    grad, wl, xl = torch.ones(256, 256, device=device), w.clone().requires_grad_(), x.clone().requires_grad_()
    version = grad._version
    y = fl.checkpointed_mlp(fl.checkpointed_linear(xl, wl, grad=grad), wl, wl, fc_grad=grad, proj_grad=grad)
    grad.zero_()
    y.backward(dy)
    assert grad._version > version + 1 and wl.grad is None
    one, got = w.clone().requires_grad_(), x.clone().requires_grad_()
    fl.checkpointed_mlp(fl.checkpointed_linear(got, one), one, one).backward(dy)
    assert torch.equal(xl.grad, got.grad)
    # three fp32 sums added in another order
    assert bool(((grad - one.grad).abs() <= 4 * EPS * (one.grad.abs() + grad.abs().max())).all())


def test_gradients_by_differences(device):
    """<gradient, v> against (L(+v) - L(-v)) / 2 of the layers without 8-bit rounding, in float64, where every value, weight and
    direction is positive: nothing cancels, so each factor's 2^-4 (and a bf16 rounding here and there) bounds the whole. dx of
    the MLP has five rounded factors (dy8, p8, sqrt(a8), dh8, f8; a8's own sums have two more, x8 and f8, under the root of a
    square), dfc and dproj no more; a value below 2^-6 of its scale's units would be off by more, so they lie within 2^10."""
    gen = torch.Generator().manual_seed(4)
    m, c, f, n = 50, 256, 384, 144
    positive = lambda *s: torch.rand(*s, generator=gen) + 0.25   # noqa: E731
    x, dy = positive(m, c).to(BF16), positive(m, n).to(BF16)
    fc, proj = positive(f, c), positive(n, f)
    xd, fd, pd = (t.to(device).requires_grad_() for t in (x, fc, proj))
    got = torch.autograd.grad(fl.checkpointed_mlp(xd, fd, pd), (xd, fd, pd), dy.to(device))

    def loss(x, fc, proj):
        return float(((x @ fc.t()).clamp(min=0).square() @ proj.t() * dy.double()).sum())

    base = [t.double() for t in (x, fc, proj)]
    bound = (1 + 2.0 ** -4) ** 7 * (1 + 2.0 ** -8) ** 3 - 1
    for i in range(3):
        v = positive(*base[i].shape).double() * 1e-3
        plus, minus = ([t + s * v if j == i else t for j, t in enumerate(base)] for s in (1, -1))
        want = (loss(*plus) - loss(*minus)) / 2
        assert abs(float((got[i].double().cpu() * v).sum()) / want - 1) <= bound
    w = fc[:n].to(device).requires_grad_()
    dx, dw = torch.autograd.grad(fl.checkpointed_linear(xd, w), (xd, w), dy.to(device))
    v = positive(m, c).double()
    assert abs(float((dx.double().cpu() * v).sum()) / float(((v @ fc[:n].double().t()) * dy.double()).sum()) - 1) <= bound
    v = positive(n, c).double()
    assert abs(float((dw.double().cpu() * v).sum()) / float(((x.double() @ v.t()) * dy.double()).sum()) - 1) <= bound


def test_gradients_of_broadcast_and_sliced_values(device):
    """A gradient without strides of its own (a sum's), transposed, misaligned or sliced, an input used twice, a frozen input
    or weight, and no rows."""
    gen = torch.Generator().manual_seed(5)
    x = bf(gen, 48, 256).to(device).requires_grad_()
    w = torch.randn(144, 256, generator=gen).to(device).requires_grad_()
    one = torch.ones(48, 144, dtype=BF16, device=device)
    want = torch.autograd.grad(fl.checkpointed_linear(x, w), (x, w), one)
    got = torch.autograd.grad(fl.checkpointed_linear(x, w).sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = bf(gen, 48, 144).to(device)
    want = torch.autograd.grad(fl.checkpointed_linear(x, w), (x, w), g)
    moved = torch.zeros(48 * 144 + 1, dtype=BF16, device=device)[1:].view(48, 144)
    moved.copy_(g)
    for other in (g.t().contiguous().t(), torch.cat([g, g], 1)[:, :144], moved):
        got = torch.autograd.grad(fl.checkpointed_linear(x, w), (x, w), other)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    y = fl.checkpointed_linear(x, w)
    twice = torch.autograd.grad((y, fl.checkpointed_linear(x, w)), w, (g, g))[0]
    assert torch.equal(twice, want[1] + want[1])
    assert torch.equal(torch.autograd.grad(fl.checkpointed_linear(x.detach(), w), w, g)[0], want[1])
    assert torch.equal(torch.autograd.grad(fl.checkpointed_linear(x, w.detach()), x, g)[0], want[0])
    fc, proj = w.detach()[:, :256].contiguous().requires_grad_(), torch.randn(32, 144, generator=gen).to(device).requires_grad_()
    empty = fl.checkpointed_mlp(x[:0], fc, proj)
    assert empty.shape == (0, 32)
    dx, dfc, dproj = torch.autograd.grad(empty, (x, fc, proj), empty.detach())
    assert not bool(dx.any()) and not bool(dfc.any()) and not bool(dproj.any())
    with pytest.raises(RuntimeError):   # no second derivative
        d = torch.autograd.grad(fl.checkpointed_linear(x, w), x, g.requires_grad_(), create_graph=True)[0]
        torch.autograd.grad(d.sum(), g)


def test_refusals_on_the_device(device):
    x, w = torch.zeros(4, 256, dtype=BF16, device=device), torch.zeros(144, 256, device=device)
    w8, (codes, scale) = fl.quantize_weight(w, True), fl.quantize_rows(x)
    for call in (lambda: fl.fp8_linear(x[:, :128], w8), lambda: fl.fp8_linear(x[:, :250], w8), lambda: fl.quantize_weight(w[0]),
                 lambda: fl.quantize_weight(w[:140], True), lambda: fl.fp8_mlp(x, w8, w8), lambda: fl.fp8_matmul(codes[:3], scale, w8),
                 lambda: fl.fp8_matmul(codes, scale.contiguous(), w8), lambda: fl.fp8_matmul(codes[:, :128], scale, w8),
                 lambda: fl.fp8_matmul(codes, scale, fl.quantize_weight(w[:137])), lambda: fl.checkpointed_linear(x, w[:140]),
                 lambda: fl.checkpointed_linear(x, w, fl.quantize_weight(w)), lambda: fl.checkpointed_linear(x, w[:128], w8),
                 lambda: fl.checkpointed_linear(x, w, grad=w[:128]), lambda: fl.checkpointed_linear(x[:, :128].contiguous(), w),
                 lambda: fl.checkpointed_mlp(x, w, w), lambda: fl.checkpoint_weight_grad(x[:3], codes, scale),
                 lambda: fl.checkpoint_weight_grad(x, codes, scale, out=w)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: fl.fp8_linear(x.float(), w8), lambda: fl.quantize_rows(x.half()), lambda: fl.quantize_weight(w.half()),
                 lambda: fl.fp8_matmul(x, scale, w8), lambda: fl.fp8_matmul(codes, scale.float(), w8),
                 lambda: fl.checkpointed_linear(x.float(), w), lambda: fl.checkpointed_linear(x, w.half()),
                 lambda: fl.checkpoint_weight_grad(x, codes, scale, dtype=torch.float16)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError, match="no backward"):
        fl.fp8_linear(x.requires_grad_(), w8)
    torch.cuda.synchronize()


def test_training_refuses_what_its_gradient_cannot_take(device):
    """Before the forward, not in the backward."""
    x, w = torch.zeros(2, 16, dtype=BF16, device=device), torch.zeros(65552, 16, dtype=BF16, device=device)
    for call in (lambda: fl.checkpointed_linear(x, w), lambda: fl.checkpointed_linear(w[:2].view(-1, 16), w),
                 lambda: fl.checkpointed_mlp(x, w, w.t().contiguous())):
        with pytest.raises(ValueError, match="65536"):
            call()
    y = fl.checkpointed_linear(x.requires_grad_(), w[:65536].requires_grad_())
    y.sum().backward()
    assert x.grad.shape == x.shape


def test_ops_give_what_their_fakes_say(device):
    """(The schema check of the same tool multiplies outputs, which torch does not do in 8 bits.)"""
    gen = torch.Generator().manual_seed(12)
    x, w, p = bf(gen, 5, 144).to(device), bf(gen, 272, 144).to(device), bf(gen, 32, 272).to(device)
    some = (None,) * 4
    utils = ("test_faketensor",)
    torch.library.opcheck(torch.ops.nanochat_amd.checkpointed_linear, (x, w, *some, None), test_utils=utils)
    torch.library.opcheck(torch.ops.nanochat_amd.checkpointed_mlp, (x, w, p, *some, None, *some, None), test_utils=utils)
    out = torch.ops.nanochat_amd.checkpointed_linear(x, w, *some, None)
    grad = torch.zeros(272, 144, device=device)
    for buffer in (None, grad):
        torch.library.opcheck(torch.ops.nanochat_amd.checkpointed_linear_bwd, (out[0], *out[1:], buffer, True, True, False),
                              test_utils=utils)


# --- together

def block(x, layers):
    """Two layers and an MLP as a model's block uses them."""
    h = fl.checkpointed_linear(x, *layers[0])
    h = x + fl.checkpointed_linear(h, *layers[1])
    return h + fl.checkpointed_mlp(h, layers[2][0], layers[3][0], layers[2][1], layers[3][1], layers[2][2], layers[3][2])


def test_training_step_captured_with_eager_work_between(device):
    """Forward and backward of a block whose weight gradients are added into fp32 buffers over two microbatches, weights
    quantized once, captured into a graph and replayed with other inputs, with eager calls of the same layers between and on
    another stream: every replay gives the eager step's bits. Then serving on the same weights."""
    gen = torch.Generator().manual_seed(6)
    shapes = [(768, 256), (256, 768), (1024, 256), (256, 1024)]
    weights = [(torch.randn(*s, generator=gen) * s[1] ** -0.5).to(device).requires_grad_() for s in shapes]
    inputs = [[bf(gen, 2, 65, 256).to(device) for _ in range(2)] for _ in range(3)]
    dys = [bf(gen, 2, 65, 256, scale=1e-2).to(device) for _ in range(3)]

    def step(xs, dy, bufs):
        layers = [(w, fl.quantize_weight(w.detach(), True), b) for w, b in zip(weights, bufs)]
        for b in bufs:
            b.zero_()
        outs = []
        for x in xs:
            x = x.detach().requires_grad_()
            y = block(x, layers)
            outs += [y.detach(), torch.autograd.grad(y, x, dy)[0]]
        return outs

    def fresh():
        return [torch.empty(*s, device=device) for s in shapes]

    want = []
    for xs, dy in zip(inputs, dys):
        bufs = fresh()
        want.append([t.clone() for t in step(xs, dy, bufs) + bufs])
    held_xs, held_dy, held_bufs = [t.clone() for t in inputs[0]], dys[0].clone(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held_xs, held_dy, held_bufs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held_xs, held_dy, held_bufs)
    for order in (0, 1, 2, 1):
        for t, s in zip(held_xs + [held_dy], inputs[order] + [dys[order]]):
            t.copy_(s)
        graph.replay()
        bufs = fresh()
        eager = step(inputs[2 - order], dys[2 - order], bufs)   # its own work between replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs + held_bufs, want[order])), order
        assert all(torch.equal(a, b) for a, b in zip(eager + bufs, want[2 - order])), order
    with torch.no_grad():
        w8 = [fl.quantize_weight(w) for w in weights]
        h = inputs[0][0] + fl.fp8_linear(fl.fp8_linear(inputs[0][0], w8[0]), w8[1])
        assert torch.equal(h + fl.fp8_mlp(h, w8[2], w8[3]), want[0][0])


@pytest.mark.parametrize("rows", [1, 12, 40, 300])
def test_serving_captured(device, rows):
    """Serving layers in a graph, replayed on new inputs with eager calls between."""
    gen = torch.Generator().manual_seed(rows)
    w, fc, proj = (weight(gen, device, *s)[0] for s in ((1296, 640), (2576, 640), (656, 2576)))
    inputs = [bf(gen, rows, 640).to(device) for _ in range(4)]
    x, s = inputs[0].clone(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fl.fp8_linear(x, w), fl.fp8_mlp(x, fc, proj)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = fl.fp8_linear(x, w), fl.fp8_mlp(x, fc, proj)
    for new in inputs[1:]:
        x.copy_(new)
        want = fl.fp8_linear(new, w), fl.fp8_mlp(new, fc, proj)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(z, want[1])


def test_two_streams_at_once(device):
    gen = torch.Generator().manual_seed(7)
    w = [weight(gen, device, 640, 1280)[0] for _ in range(2)]
    x = [bf(gen, 300, 1280).to(device) for _ in range(2)]
    want = [fl.fp8_linear(a, b) for a, b in zip(x, w)]
    grads = [fl.checkpoint_weight_grad(y, *fl.quantize_rows(a)) for y, a in zip(want, x)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, a, b in zip(streams, x, w):
            with torch.cuda.stream(s):
                y = fl.fp8_linear(a, b)
                got.append((y, fl.checkpoint_weight_grad(y, *fl.quantize_rows(a))))
        torch.cuda.synchronize()
        assert all(torch.equal(y, t) and torch.equal(g, u) for (y, g), t, u in zip(got, want, grads))


def test_more_than_two_to_the_31_bytes(device):
    """Rows whose codes and results lie past 2^31 bytes, first and last rows alike."""
    gen = torch.Generator().manual_seed(8)
    few, rows, k, n = bf(gen, 300, 1024).to(device), 2 ** 21 + 300, 1024, 1040
    x = few.repeat(-(-rows // 300), 1)[:rows].contiguous()
    w, _ = weight(gen, device, n, k)
    codes, scale = fl.quantize_rows(x)
    y = fl.fp8_matmul(codes, scale, w)
    first = fl.fp8_matmul(*fl.quantize_rows(few), w)
    last = torch.arange(rows - 300, rows, device=device)
    assert torch.equal(y[last], first[last % 300]) and torch.equal(codes[last].view(torch.uint8), codes[last % 300].view(torch.uint8))
    dw = fl.checkpoint_weight_grad(y[:, :64].contiguous(), codes, scale)
    part = few.double()[torch.arange(300, device=device)]
    x8 = torch.from_numpy(fb.through(part.cpu().numpy(), 1)).to(device)
    counts = torch.bincount(torch.arange(rows, device=device) % 300, minlength=300).double()
    want = (first[:, :64].double() * counts[:, None]).t() @ x8
    mag = (first[:, :64].double().abs() * counts[:, None]).t() @ x8.abs()
    assert bool(((dw.double() - want).abs() <= 2.0 ** -12 * mag).all())   # fp32 sums of at most 8,192 rows a slice and 256 slices
