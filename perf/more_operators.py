"""Products in 8-bit floating point and the training of linear layers from 8-bit checkpoints of their inputs, in their
plain form and as this framework offers them.

- listed()            named cases: the smallest calls, ordinary ones, the largest
- draw(rng)           one more case of the same ranges
- prepare(case, seed) what a program holds before the call: its inputs and weights
- run(state)          one pass; with `own` false in elementary torch operations, else through nanochat_amd
- work(case)          bytes and flops one pass cannot do without
- exact(case, seed)   run's outputs from the definitions, in float64

The 8-bit form of a matrix: e4m3 codes and one power of two for each block, the least s with max |x| <= 448 s (1 for a
block of zeros), a value standing for code times s. Blocks are 128 columns of a row of activations or gradients, and 128 x
128 of a weight; the last of a row or column may be shorter. A power of two costs nothing (e4m3 is as exact at any scale,
until it runs out of exponents) and makes a value exact in bf16.

Kinds of case:

  linear        y = x8 w8^T, bf16 in and out: x8 the 8-bit form of x's rows, w8 a weight held in 8 bits
                (fp8_linear.fp8_linear)
  mlp           y = a8 p8^T with a = relu(x8 f8^T)^2, its two weights held in 8 bits (fp8_linear.fp8_mlp)
  train_linear  the same product in training, from a bf16 or fp32 weight, and its gradients. x8 is all that is kept of x:
                dx = dy8 w8, dw = dy^T x8 (fp8_linear.checkpointed_linear)
  train_mlp     the MLP in training: x8 and a8 are all that is kept. da = dy8 p8, dh = bf16(2 sqrt(a8) da), dx = dh8 f8,
                df = dh^T x8, dp = dy^T a8 (fp8_linear.checkpointed_mlp)
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 128
FP8_MAX = 448.0


def listed():
    return [
        # One user's next token through the fused q, k, v projection of the 13-head model. Latency is all.
        dict(name="linear_one", kind="linear", rows=1, inner=1664, outer=4992),
        # A few draft tokens of several users, no round number, the 10-head model's square projection.
        dict(name="linear_few", kind="linear", rows=37, inner=1280, outer=1280),
        # The logits of a full batch of 128 slots: the widest weight of all, read once.
        dict(name="linear_head", kind="linear", rows=128, inner=1664, outer=65536),
        # Prompt chunks of eight requests at once: bound by the matrix cores.
        dict(name="linear_prompts", kind="linear", rows=16384, inner=1664, outer=4992),
        # One token through the 13-head model's MLP.
        dict(name="mlp_one", kind="mlp", rows=1, inner=1664, hidden=6656),
        # A decoding batch.
        dict(name="mlp_batch", kind="mlp", rows=128, inner=1664, hidden=6656),
        # Prompts of odd lengths, packed, in the 10-head model.
        dict(name="mlp_prompts", kind="mlp", rows=9995, inner=1280, hidden=5120),
        # A short microbatch of the 6-head model's square projection with an fp32 master weight.
        dict(name="train_linear_short", kind="train_linear", rows=515, inner=768, outer=768, weight="float32"),
        # A training step's tokens (32 x 2,048) through the q, k, v projection.
        dict(name="train_linear_step", kind="train_linear", rows=65536, inner=1664, outer=4992, weight="float32"),
        # A fine-tuning batch of a few documents, packed, bf16 weights.
        dict(name="train_mlp_short", kind="train_mlp", rows=1001, inner=1280, hidden=5120, weight="bfloat16"),
        # A quarter of a step's tokens, as one of four microbatches.
        dict(name="train_mlp_micro", kind="train_mlp", rows=16384, inner=1280, hidden=5120, weight="bfloat16"),
        # A training step's tokens through the 13-head model's MLP: the largest.
        dict(name="train_mlp_step", kind="train_mlp", rows=65536, inner=1664, hidden=6656, weight="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_linear(rng):
    inner, outer = 16 * _log_int(rng, 4, 512), 16 * _log_int(rng, 4, 1024)
    rows = _log_int(rng, 1, 16384)
    while rows * inner * outer > 16384 * 1664 * 6656:
        rows = max(1, rows * 3 // 4)
    return dict(kind="linear", rows=rows, inner=inner, outer=outer)


def _draw_mlp(rng):
    inner = 16 * _log_int(rng, 8, 160)
    hidden = rng.choice([4 * inner, 16 * _log_int(rng, 16, 640)])
    rows = _log_int(rng, 1, 16384)
    while rows * inner * hidden > 16384 * 1664 * 6656:
        rows = max(1, rows * 3 // 4)
    return dict(kind="mlp", rows=rows, inner=inner, hidden=hidden)


def _draw_train_linear(rng):
    inner, outer = 16 * _log_int(rng, 8, 320), 16 * _log_int(rng, 8, 320)
    return dict(kind="train_linear", rows=_log_int(rng, 16, 32768), inner=inner, outer=outer,
                weight=rng.choice(["float32", "bfloat16"]))


def _draw_train_mlp(rng):
    inner = 16 * _log_int(rng, 8, 128)
    return dict(kind="train_mlp", rows=_log_int(rng, 16, 32768), inner=inner,
                hidden=rng.choice([4 * inner, 16 * _log_int(rng, 16, 400)]), weight="bfloat16")


def draw(rng):
    return rng.choice([_draw_linear, _draw_mlp, _draw_train_linear, _draw_train_mlp])(rng)


def work(case):
    m, k = case["rows"], case["inner"]
    n = case["outer"] if "outer" in case else case["hidden"]
    if case["kind"] == "linear":
        return {"bytes": 2 * m * (k + n) + n * k, "flops": 2 * m * n * k}
    if case["kind"] == "mlp":
        return {"bytes": 4 * m * k + 2 * n * k, "flops": 4 * m * n * k}
    wide = 4 if case["weight"] == "float32" else 2
    if case["kind"] == "train_linear":   # x, w, dy in; y, dx, dw out
        return {"bytes": 4 * m * (k + n) + 2 * wide * n * k, "flops": 6 * m * n * k}
    return {"bytes": 8 * m * k + 4 * wide * n * k, "flops": 12 * m * n * k}   # x, dy, both weights in; y, dx, theirs out


# --- the 8-bit form, plain

def _scale(amax):
    """The least power of two s with amax <= 448 s, 1 for 0."""
    fraction, exponent = torch.frexp(amax)                    # amax = fraction 2^exponent, fraction in [0.5, 1)
    exponent = exponent - 9 + (fraction > FP8_MAX / 512).to(exponent.dtype)
    exponent = torch.where(amax > 0, exponent, 0).clamp(-126, 127)
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.size(1) % cols, 0, -x.size(0) % rows))


def _blocks(x, rows):
    """fp32 [R, C] as [blocks of `rows` rows, rows, blocks of 128 columns, 128], zeros past its edges."""
    x = _padded(x, rows, BLOCK)
    return x.view(x.size(0) // rows, rows, x.size(1) // BLOCK, BLOCK)


def _codes(x, rows):
    """(e4m3 codes like x, fp32 scales [blocks of rows, blocks of columns])."""
    b = _blocks(x.float(), rows)
    scale = _scale(b.abs().amax((1, 3)))
    codes = (b / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.flatten(2).flatten(0, 1)[:x.size(0), :x.size(1)].contiguous(), scale


def _values(codes, scale, rows):
    """The fp32 values that codes stand for."""
    return (_blocks(codes.float(), rows) * scale[:, None, :, None]).flatten(2).flatten(0, 1)[
        :codes.size(0), :codes.size(1)]


def _through(x, rows):
    """x (rounded to 8 bits), as fp32 values."""
    return _values(*_codes(x, rows), rows)


# --- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _activations(gen, rows, cols):
    """bf16 rows of sizes of their own, a few channels far above the others, as a normed residual stream has them."""
    x = torch.randn(rows, cols, generator=gen, device=DEVICE)
    channel = torch.exp(0.5 * torch.randn(cols, generator=gen, device=DEVICE))
    loud = torch.rand(cols, generator=gen, device=DEVICE) < 0.01
    x *= torch.where(loud, 10 * channel, channel) * torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device=DEVICE))
    return x.to(torch.bfloat16)


def _weight(gen, outer, inner, dtype=torch.float32):
    w = torch.randn(outer, inner, generator=gen, device=DEVICE)
    return (w * inner ** -0.5 * torch.exp(0.2 * torch.randn(outer, 1, generator=gen, device=DEVICE))).to(dtype)


def _gradient(gen, rows, cols):
    """bf16 rows of a mean loss's gradient: small, and over a few powers of two from token to token."""
    g = torch.randn(rows, cols, generator=gen, device=DEVICE)
    g *= torch.exp(torch.randn(rows, 1, generator=gen, device=DEVICE)) / rows
    return g.to(torch.bfloat16)


def _held(w):
    """A weight as a serving program holds it: codes and, in bytes of exponents, scales, their rows 4-byte aligned."""
    codes, scale = _codes(w, BLOCK)
    held = torch.zeros(scale.size(0), -(-scale.size(1) // 4) * 4, dtype=torch.uint8, device=DEVICE)
    held[:, :scale.size(1)] = (scale.view(torch.int32) >> 23).to(torch.uint8)
    return dict(codes=codes, scale=held.view(torch.float8_e8m0fnu)[:, :scale.size(1)])


def prepare(case, seed):
    gen, kind = _generator(seed), case["kind"]
    m, k = case["rows"], case["inner"]
    s = dict(case=dict(case), x=_activations(gen, m, k))
    if kind == "linear":
        s["w"] = _held(_weight(gen, case["outer"], k))
    elif kind == "mlp":
        s["fc"], s["proj"] = _held(_weight(gen, case["hidden"], k)), _held(_weight(gen, k, case["hidden"]))
    else:
        dtype = getattr(torch, case["weight"])
        shapes = [(case["outer"], k)] if kind == "train_linear" else [(case["hidden"], k), (k, case["hidden"])]
        s["weights"] = [_weight(gen, *shape, dtype).requires_grad_() for shape in shapes]
        s["dy"] = _gradient(gen, m, shapes[-1][0])
        s["x"].requires_grad_()
    return s


# --- the plain forms

def _dequantized(w):
    return _values(w["codes"], (w["scale"].view(torch.uint8).to(torch.int32) << 23).view(torch.float32), BLOCK)


def _plain_linear(s):
    return (_through(s["x"], 1) @ _dequantized(s["w"]).t()).to(torch.bfloat16)


def _plain_mlp(s):
    h = _through(s["x"], 1) @ _dequantized(s["fc"]).t()
    return (_through(h.clamp_(min=0).square_(), 1) @ _dequantized(s["proj"]).t()).to(torch.bfloat16)


def _plain_train_linear(s):
    (w,), x, dy = s["weights"], _through(s["x"], 1), s["dy"]
    w8 = _through(w, BLOCK)
    return dict(y=(x @ w8.t()).to(torch.bfloat16), dx=(_through(dy, 1) @ w8).to(torch.bfloat16),
                dw=(dy.float().t() @ x).to(w.dtype))


def _plain_train_mlp(s):
    (fc, proj), x, dy = s["weights"], _through(s["x"], 1), s["dy"]
    f8, p8 = _through(fc, BLOCK), _through(proj, BLOCK)
    a = _through((x @ f8.t()).clamp_(min=0).square_(), 1)
    y = (a @ p8.t()).to(torch.bfloat16)
    dh = (_through(dy, 1) @ p8).mul_(a.sqrt().mul_(2)).to(torch.bfloat16)
    return dict(y=y, dx=(_through(dh, 1) @ f8).to(torch.bfloat16), dfc=(dh.float().t() @ x).to(fc.dtype),
                dproj=(dy.float().t() @ a).to(proj.dtype))


# --- the framework's

def _own_linear(s):
    from nanochat_amd.fp8_linear import Fp8Weight, fp8_linear

    return fp8_linear(s["x"], Fp8Weight(**s["w"]))


def _own_mlp(s):
    from nanochat_amd.fp8_linear import Fp8Weight, fp8_mlp

    return fp8_mlp(s["x"], Fp8Weight(**s["fc"]), Fp8Weight(**s["proj"]))


def _own_train_linear(s):
    from nanochat_amd.fp8_linear import checkpointed_linear

    (w,) = s["weights"]
    y = checkpointed_linear(s["x"], w)
    dx, dw = torch.autograd.grad(y, (s["x"], w), s["dy"])
    return dict(y=y, dx=dx, dw=dw)


def _own_train_mlp(s):
    from nanochat_amd.fp8_linear import checkpointed_mlp

    fc, proj = s["weights"]
    y = checkpointed_mlp(s["x"], fc, proj)
    dx, dfc, dproj = torch.autograd.grad(y, (s["x"], fc, proj), s["dy"])
    return dict(y=y, dx=dx, dfc=dfc, dproj=dproj)


PLAIN = dict(linear=_plain_linear, mlp=_plain_mlp, train_linear=_plain_train_linear, train_mlp=_plain_train_mlp)
OWN = dict(linear=_own_linear, mlp=_own_mlp, train_linear=_own_train_linear, train_mlp=_own_train_mlp)


def run(state):
    if own:
        return OWN[state["case"]["kind"]](state)
    with torch.no_grad():
        return PLAIN[state["case"]["kind"]](state)


# --- the definitions in float64

def _rounded8(x, rows):
    """float64 x to the nearest value of its block's 8-bit form, ties to even: a step is 2^-3 of the value's power of two
    (2^-9 below 2^-6), in units of the block's scale."""
    r, c = x.shape
    full = torch.zeros(-(-r // rows) * rows, -(-c // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:r, :c] = x
    b = full.reshape(-(-r // rows), rows, -(-c // BLOCK), BLOCK)
    most = b.abs().amax(dim=(1, 3), keepdim=True)
    power = torch.ceil(torch.log2(torch.where(most > 0, most, FP8_MAX) / FP8_MAX))
    power = torch.where(FP8_MAX * torch.exp2(power) < most, power + 1, power)          # log2's own error
    power = torch.where((FP8_MAX * torch.exp2(power - 1) >= most) & (most > 0), power - 1, power)
    unit = torch.exp2(power)                                                            # of whole numbers: exact
    b = b / unit
    size = torch.frexp(b)[1] - 1
    step = torch.exp2((size.clamp(min=-6) - 3).double())
    return (torch.round(b / step) * step * unit).reshape(full.shape)[:r, :c]


def _held64(w):
    power = (w["scale"].view(torch.uint8).double() - 127).repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
    n, k = w["codes"].shape
    return w["codes"].double() * torch.exp2(power[:n, :k])


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    with torch.no_grad():
        x = _rounded8(s["x"].double(), 1)
        if kind == "linear":
            return x @ _held64(s["w"]).t()
        if kind == "mlp":
            h = x @ _held64(s["fc"]).t()
            return _rounded8(torch.where(h > 0, h * h, 0.0), 1) @ _held64(s["proj"]).t()
        weights, dy = [_rounded8(w.double(), BLOCK) for w in s["weights"]], s["dy"].double()
        dy8 = _rounded8(dy, 1)
        if kind == "train_linear":
            return dict(y=x @ weights[0].t(), dx=dy8 @ weights[0], dw=dy.t() @ x)
        fc, proj = weights
        h = x @ fc.t()
        a = _rounded8(torch.where(h > 0, h * h, 0.0), 1)
        del h
        y = a @ proj.t()
        dproj = dy.t() @ a
        dh = ((dy8 @ proj) * (2 * a.sqrt())).to(torch.bfloat16).double()
        del a
        return dict(y=y, dx=_rounded8(dh, 1) @ fc, dfc=dh.t() @ x, dproj=dproj)
