"""Linear layers in 8-bit floating point, and their training from 8-bit checkpoints of their inputs (csrc/fp8_quant.hip,
fp8_gemm.hip, fp8_grad.hip). No counterpart in the reference, whose linear layers and ReLU^2 MLP are bf16
(model/ops/linear.py:51-57, 135-144).

The 8-bit form of a matrix: e4m3 codes and one power of two for each block, held as its exponent (torch.float8_e8m0fnu).
Blocks are 128 columns of a row of activations or gradients and 128 x 128 of a weight. The scale is the least s with
max |x| <= 448 s; a code stands for code * s. A power of two makes that value exact in bf16 and lets the matrix cores apply
the scales themselves. A block that holds an infinity or a NaN becomes NaN whole.

- quantize_rows, quantize_weight: the 8-bit form of activations, of weights (with that of the transpose, for training)
- fp8_linear, fp8_mlp: a layer, and a ReLU^2 MLP, on weights held in 8 bits, for serving: one row to many thousand
- fp8_matmul: the product of activations already in 8 bits
- checkpointed_linear, checkpointed_mlp: the same in training, over the registered ops nanochat_amd::checkpointed_linear[_bwd] and
  nanochat_amd::checkpointed_mlp[_bwd]. What is kept for the backward is the 8-bit form of the layer's input (and of the MLP's
  hidden activations): half of bf16's bytes, and the very operand that the forward product took
- checkpoint_weight_grad: a weight's gradient from such a checkpoint

Every function launches on the current stream of its input's device and requires device tensors: there is no CPU path."""

from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd.function import FunctionCtx, once_differentiable

from .native import check, device_guard, hip_library, pointer, stream

BLOCK = 128
CODES, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
BF16, F32 = torch.bfloat16, torch.float32
MOST = 65536   # a weight's rows and columns in training, as its gradient's kernel has them


class Fp8Weight(NamedTuple):
    """A weight [N, K] in the 8-bit form: codes [N, K], scale [ceil(N / 128), ceil(K / 128)] (rows at a stride that is a
    multiple of 4), and for training those of its transpose, codes_t [K, N] and scale_t."""
    codes: Tensor
    scale: Tensor
    codes_t: Tensor | None = None
    scale_t: Tensor | None = None


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _new_scale(like: Tensor, rows: int, cols: int) -> Tensor:
    """Scales [rows, ceil(cols / 128)], their rows padded to a multiple of 4 bytes."""
    blocks = _blocks(cols)
    return torch.empty(rows, -(-blocks // 4) * 4, dtype=SCALE, device=like.device)[:, :blocks]


def _check_codes(codes: Tensor, name: str, device: torch.device, part: str = "") -> None:
    if codes.dtype != CODES:
        raise TypeError(f"{name}{part} must be {CODES}, got {codes.dtype}")
    if codes.device != device or not codes.is_cuda:
        raise ValueError(f"{name}{part} must be a device tensor on {device}, got {codes.device}")
    if codes.dim() != 2 or not codes.is_contiguous() or codes.data_ptr() % 16:
        raise ValueError(f"{name}{part} must be a contiguous, 16-byte aligned matrix")
    if codes.size(1) % 16:
        raise ValueError(f"{name}{part} must have a multiple of 16 columns, got {codes.size(1)}")


def _check_scale(scale: Tensor, name: str, rows: int, cols: int, device: torch.device, part: str = "",
                 padded: bool = False) -> int:
    """A scale tensor's row stride in bytes. padded: it may have its rows' padding in its shape, as an op returns it."""
    if scale.dtype != SCALE:
        raise TypeError(f"{name}{part} must be {SCALE}, got {scale.dtype}")
    blocks = -(-cols // BLOCK)
    if (scale.dim() != 2 or scale.device != device
            or (scale.shape != (rows, blocks) and not (padded and scale.shape == (rows, -(-blocks // 4) * 4)))):
        raise ValueError(f"{name}{part} must be [{rows}, {blocks}] on {device}, got {tuple(scale.shape)} on {scale.device}")
    pitch, step = scale.stride()
    if ((blocks > 1 and step != 1) or pitch % 4 or pitch < blocks or pitch > cols or scale.data_ptr() % 4
            or scale.storage_offset() + (rows - 1) * pitch + -(-blocks // 4) * 4 > scale.untyped_storage().nbytes()):
        raise ValueError(f"{name}{part} must have 4-byte aligned rows of adjacent scales, padded to a multiple of 4 bytes")
    return pitch


def _check_weight(w: Fp8Weight, name: str, device: torch.device, transposed: bool = False) -> tuple[int, int]:
    """(pitch of the scales, of the transpose's or 0) of a weight in the 8-bit form."""
    codes, scale, codes_t, scale_t = w
    _check_codes(codes, name, device, ".codes")
    n, k = codes.shape
    pitch = _check_scale(scale, name, -(-n // BLOCK), k, device, ".scale")
    if not transposed:
        return pitch, 0
    if codes_t is None or scale_t is None:
        raise ValueError(f"{name} needs its transpose for training: quantize_weight(w, transpose=True)")
    _check_codes(codes_t, name, device, ".codes_t")
    if codes_t.shape != (k, n):
        raise ValueError(f"{name}.codes_t must be {(k, n)}, got {tuple(codes_t.shape)}")
    return pitch, _check_scale(scale_t, name, -(-k // BLOCK), n, device, ".scale_t")


def _check_kept(codes: Tensor, scale: Tensor, names: tuple[str, str], rows: int, cols: int, of: int, device: torch.device) -> None:
    """An 8-bit form as a backward op is given it: codes [rows, cols] with a scale for each `of` rows."""
    # as the forward ops return it, in one expression (1.6 us; the checks below, which say what is wrong, 3 to 4)
    if (codes.dtype == CODES and scale.dtype == SCALE and codes.shape == (rows, cols) and codes.device == device == scale.device
            and scale.shape == (-(-rows // of), -(-cols // (4 * BLOCK)) * 4) and codes.is_contiguous() and scale.is_contiguous()
            and codes.is_cuda and not (cols % 16 or codes.data_ptr() % 16 or scale.data_ptr() % 4)):
        return
    _check_codes(codes, names[0], device)
    if codes.shape != (rows, cols):
        raise ValueError(f"{names[0]} must be {(rows, cols)}, got {tuple(codes.shape)}")
    _check_scale(scale, names[1], -(-rows // of), cols, device, padded=True)


def _as_rows(x: Tensor, name: str, dtypes: tuple, of: int = 16) -> Tensor:
    """x as rows [M, K] of adjacent values that do not overlap: a view where there is one."""
    if not x.is_cuda:
        raise ValueError(f"{name} must be a device tensor (the 8-bit layers have no CPU implementation)")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(map(str, dtypes))}, got {x.dtype}")
    if x.dim() < 1 or x.size(-1) < 1 or x.size(-1) % of:
        raise ValueError(f"{name} must have a multiple of {of} columns, got {tuple(x.shape)}")
    if x.dim() != 2:
        x = x.reshape(-1, x.size(-1))
    if x.stride(1) != 1 or (x.size(0) > 1 and x.stride(0) < x.size(1)):
        x = x.contiguous()
    return x


def _quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    rows, cols = x.shape
    codes, scale = torch.empty(rows, cols, dtype=CODES, device=x.device), _new_scale(x, rows, cols)
    if rows:
        check(hip_library().nc_fp8_quantize_rows(pointer(x), x.dtype == F32, x.stride(0) if rows > 1 else cols, rows, cols,
                                                 pointer(codes), pointer(scale), scale.stride(0), stream()))
    return codes, scale


def quantize_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    """x bf16 or fp32 [..., K] (K a multiple of 16; rows of any stride, others are copied) -> its 8-bit form: codes
    e4m3 [rows, K], scale e8m0 [rows, ceil(K / 128)], rows being all leading dimensions."""
    x = _as_rows(x, "x", (BF16, F32))
    with device_guard(x):
        return _quantize(x)


def quantize_weight(w: Tensor, transpose: bool = False) -> Fp8Weight:
    """A weight bf16 or fp32 [N, K], K (and N with its transpose) a multiple of 16 -> its 8-bit form."""
    if w.dim() != 2:
        raise ValueError(f"w must be [N, K], got {tuple(w.shape)}")
    w = _as_rows(w, "w", (BF16, F32))
    n, k = w.shape
    if n < 1 or (transpose and n % 16):
        raise ValueError(f"w must have rows{', a multiple of 16 for its transpose' if transpose else ''}, got {n}")
    codes, scale = torch.empty(n, k, dtype=CODES, device=w.device), _new_scale(w, _blocks(n), k)
    codes_t = scale_t = None
    if transpose:
        codes_t, scale_t = torch.empty(k, n, dtype=CODES, device=w.device), _new_scale(w, _blocks(k), n)
    with device_guard(w):
        check(hip_library().nc_fp8_quantize_weight(
            pointer(w), w.dtype == F32, w.stride(0) if n > 1 else k, n, k, pointer(codes), pointer(scale), scale.stride(0),
            pointer(codes_t) if transpose else None, pointer(scale_t) if transpose else None,
            scale_t.stride(0) if transpose else 0, stream()))
    return Fp8Weight(codes, scale, codes_t, scale_t)


def _product(codes: Tensor, scale: Tensor, w_codes: Tensor, w_scale: Tensor) -> Tensor:
    rows, k = codes.shape
    n = w_codes.size(0)
    out = torch.empty(rows, n, dtype=BF16, device=codes.device)
    check(hip_library().nc_fp8_matmul(pointer(codes), pointer(scale), scale.stride(0), pointer(w_codes), pointer(w_scale),
                                      w_scale.stride(0), rows, n, k, pointer(out), stream()))
    return out


def _outputs(n: int, name: str) -> None:
    if n % 16:
        raise ValueError(f"{name} must have a multiple of 16 rows for a product, got {n}")


def fp8_matmul(codes: Tensor, scale: Tensor, weight: Fp8Weight) -> Tensor:
    """Activations in the 8-bit form (quantize_rows') [M, K] times a weight's transpose: bf16 [M, N], N and K multiples of
    16. Sums are fp32, but for the eight products of adjacent columns that the matrix cores add at a time: of those, bits
    below 2^-13 of the largest are dropped (at most 2^-10 of the sum of magnitudes; 1e-5 to 3e-5 of a result as a rule)."""
    device = codes.device
    _check_codes(codes, "codes", device)
    _check_scale(scale, "scale", codes.size(0), codes.size(1), device)
    _check_weight(weight, "weight", device)
    if weight.codes.size(1) != codes.size(1):
        raise ValueError(f"codes have {codes.size(1)} columns, the weight {weight.codes.size(1)}")
    _outputs(weight.codes.size(0), "weight")
    with device_guard(codes):
        return _product(codes, scale, weight.codes, weight.scale)


def _serving_input(x: Tensor, weight: Fp8Weight, name: str) -> Tensor:
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} has no backward: use checkpointed_linear or checkpointed_mlp, or torch.no_grad()")
    rows = _as_rows(x, "x", (BF16,))
    if weight.codes.dim() != 2 or weight.codes.size(1) != rows.size(1):
        raise ValueError(f"x has {rows.size(1)} columns for a weight of {tuple(weight.codes.shape)}")
    return rows


FEW = 64          # rows that one launch of the few-row kernel takes
NO_POINTER = -1   # a call's status where a pointer that it needs is missing (NC_ERR_NULL)


def _workspace(x: Tensor, need: int) -> Tensor:
    return torch.empty(max(need, 16), dtype=torch.uint8, device=x.device)   # an unsupported size: refused by the call


def fp8_linear(x: Tensor, weight: Fp8Weight) -> Tensor:
    """x bf16 [..., K] through a linear layer whose weight [N, K] is held in 8 bits: bf16 [..., N]. Each row of x is taken in
    its 8-bit form. For serving: no gradient (checkpointed_linear has one)."""
    rows = _serving_input(x, weight, "fp8_linear")
    pitch, _ = _check_weight(weight, "weight", x.device)
    (m, k), n = rows.shape, weight.codes.size(0)
    _outputs(n, "weight")
    with device_guard(x):
        call, at, stride = hip_library().nc_fp8_linear, rows.data_ptr(), rows.stride(0)
        out = torch.empty(m, n, dtype=BF16, device=x.device)
        args = (at, 0, stride, weight.codes.data_ptr(), weight.scale.data_ptr(), pitch, m, n, k, out.data_ptr())
        # a few rows need no workspace as a rule: asked for only where the call refuses to go without
        status = call(*args, None, 0, stream()) if m <= FEW else NO_POINTER
        if status == NO_POINTER:
            need = hip_library().nc_fp8_linear_workspace_bytes(at, 0, stride, m, n, k)
            ws = _workspace(x, need)
            status = call(*args, ws.data_ptr(), need, stream())
        check(status)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], n)


def fp8_mlp(x: Tensor, fc: Fp8Weight, proj: Fp8Weight, fast: bool = False) -> Tensor:
    """x bf16 [..., C] through proj(relu(fc(x))^2), fc [F, C] and proj [N, F] held in 8 bits: bf16 [..., N]. The squared
    activations are taken in their 8-bit form from fp32 sums of exact products. fast: for many rows (ceil(rows / 64) ceil(F / 128)
    above the number of CUs) that product takes 0.55 to 0.6 of the time, and drops bits as fp8_matmul's does: some 5 of 10,000 squares, which
    lie on the border of two codes, then get the other one, and a result lies 0.0024 to 0.0037 (relative norm) from what float64
    makes of the same operands, in place of the 0.0017 that its own rounding to bf16 makes (the 8-bit form itself puts it 0.057 off the
    MLP without it). For serving: no gradient (checkpointed_mlp has one)."""
    rows = _serving_input(x, fc, "fp8_mlp")
    fc_pitch, _ = _check_weight(fc, "fc", x.device)
    proj_pitch, _ = _check_weight(proj, "proj", x.device)
    (m, c), (n, hidden) = rows.shape, proj.codes.shape
    if hidden != fc.codes.size(0):
        raise ValueError(f"proj {tuple(proj.codes.shape)} does not take fc's {fc.codes.size(0)} outputs")
    _outputs(n, "proj")
    with device_guard(x):
        lib = hip_library()
        need = lib.nc_fp8_mlp_workspace_bytes(m, c, hidden)
        out, ws = torch.empty(m, n, dtype=BF16, device=x.device), _workspace(x, need)
        call = lib.nc_fp8_mlp_fast if fast else lib.nc_fp8_mlp
        check(call(rows.data_ptr(), rows.stride(0), fc.codes.data_ptr(), fc.scale.data_ptr(), fc_pitch, proj.codes.data_ptr(),
                   proj.scale.data_ptr(), proj_pitch, m, c, hidden, n, out.data_ptr(), ws.data_ptr(), need, stream()))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], n)


# --- training

_GRAD_NONE, _GRAD_F32, _GRAD_ADD, _GRAD_BF16 = -1, 0, 1, 2


def _weight_grad(dy: Tensor, codes: Tensor, scale: Tensor, out: Tensor, mode: int) -> Tensor:
    (rows, n1), n2 = dy.shape, codes.size(1)
    if rows == 0:
        return out if mode == _GRAD_ADD else out.zero_()
    lib = hip_library()
    need = lib.nc_fp8_weight_grad_workspace_bytes(rows, n1, n2)
    ws = _workspace(dy, need)
    check(lib.nc_fp8_weight_grad(pointer(dy), pointer(codes), pointer(scale), scale.stride(0), rows, n1, n2, mode,
                                 pointer(out), pointer(ws), need, stream()))
    return out


def _dense(t: Tensor) -> Tensor:
    """t [M, N] with its rows one after another from a 16-byte border, as the weight gradient reads them."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_grad(grad: Tensor, shape: tuple, device: torch.device, name: str) -> None:
    if grad.dtype != F32 or grad.device != device:
        raise ValueError(f"{name} must be {F32} on {device}, got {grad.dtype} on {grad.device}")
    if tuple(grad.shape) != tuple(shape) or not grad.is_contiguous() or grad.data_ptr() % 16:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned {tuple(shape)}, got {tuple(grad.shape)}")


def _written(t: Tensor) -> None:
    """t is added to in place: autograd may hold it for a backward of its own, which has to notice."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def checkpoint_weight_grad(dy: Tensor, codes: Tensor, scale: Tensor, out: Tensor | None = None,
                           dtype: torch.dtype = F32) -> Tensor:
    """The gradient dy^T x of a weight [N, K], dy bf16 [..., N] (N a multiple of 8) the gradient behind the layer and x [M, K] the 8-bit
    checkpoint of its input (quantize_rows'). Products are exact and sums fp32; the result is fp32, or rounded once to bf16
    (dtype), or added to out (fp32 [N, K]) when given."""
    dy = _as_rows(dy, "dy", (BF16,), of=8)
    _check_codes(codes, "codes", dy.device)
    _check_scale(scale, "scale", codes.size(0), codes.size(1), dy.device)
    if dy.size(0) != codes.size(0):
        raise ValueError(f"dy has {dy.size(0)} rows, the checkpoint {codes.size(0)}")
    shape = (dy.size(1), codes.size(1))
    if out is not None:
        _check_grad(out, shape, dy.device, "out")
        _written(out)
    elif dtype not in (F32, BF16):
        raise TypeError(f"dtype must be {F32} or {BF16}, got {dtype}")
    with device_guard(dy):
        if out is not None:
            return _weight_grad(_dense(dy), codes, scale, out, _GRAD_ADD)
        out = torch.empty(shape, dtype=dtype, device=dy.device)
        return _weight_grad(_dense(dy), codes, scale, out, _GRAD_F32 if dtype == F32 else _GRAD_BF16)


def _held(weight: Tensor, name: str, codes: Tensor | None, scale: Tensor | None, codes_t: Tensor | None,
          scale_t: Tensor | None, grad: Tensor | None, device: torch.device) -> tuple[Tensor, Tensor, int, Tensor, Tensor]:
    """A layer's arguments checked -> codes, scales and their pitch in the 8-bit form that its op uses, then what its backward
    reads: from what it was given (that then empty, as the caller holds it), or the weight's own form, made now."""
    if weight.dim() != 2 or weight.size(0) % 16 or weight.size(1) % 16 or weight.numel() == 0 or max(weight.shape) > MOST:
        raise ValueError(f"{name} must be [N, K], both multiples of 16 up to {MOST}, got {tuple(weight.shape)}")
    if weight.dtype not in (BF16, F32):
        raise TypeError(f"{name} must be {BF16} or {F32}, got {weight.dtype}")
    if weight.device != device:
        raise ValueError(f"{name} must be on {device}, got {weight.device}")
    if grad is not None:
        _check_grad(grad, weight.shape, device, f"{name}'s gradient")
    n, k = weight.shape
    if codes is not None:
        pitch, _ = _check_weight(Fp8Weight(codes, scale, codes_t, scale_t), f"{name} in 8 bits", device, transposed=True)
        if codes.shape != (n, k):
            raise ValueError(f"{name} is {(n, k)}, its 8-bit form {tuple(codes.shape)}")
        return codes, scale, pitch, codes.new_empty(0), scale.new_empty(0)
    w = _as_rows(weight, name, (BF16, F32))
    codes, scale = torch.empty(n, k, dtype=CODES, device=device), _whole_scale(w, _blocks(n), k)
    codes_t, scale_t = torch.empty(k, n, dtype=CODES, device=device), _whole_scale(w, _blocks(k), n)
    pitch = scale.size(1)
    check(hip_library().nc_fp8_quantize_weight(w.data_ptr(), w.dtype == F32, w.stride(0), n, k, codes.data_ptr(),
                                               scale.data_ptr(), pitch, codes_t.data_ptr(), scale_t.data_ptr(),
                                               scale_t.size(1), stream()))
    return codes, scale, pitch, codes_t, scale_t


def _whole_scale(like: Tensor, rows: int, cols: int) -> Tensor:
    """New scales with their rows' padding, as an op returns them."""
    return torch.empty(rows, -(-_blocks(cols) // 4) * 4, dtype=SCALE, device=like.device)


def _layer_grad(weight: int, k: int, grad: Tensor | None, wanted: bool, wide: bool, like: Tensor,
                name: str) -> tuple[Tensor, int, Tensor]:
    """A layer's weight gradient [weight, k] as its op returns it (new, or empty where it goes into grad or is not wanted), the
    mode that makes it, and where it goes. grad is checked here, where it is written: since the forward it may have changed."""
    if not wanted:
        return like.new_empty(0), _GRAD_NONE, None
    if grad is not None:
        _check_grad(grad, (weight, k), like.device, name)
        _written(grad)
        return like.new_empty(0), _GRAD_ADD, grad
    out = torch.empty(weight, k, dtype=F32 if wide else BF16, device=like.device)
    return out, _GRAD_F32 if wide else _GRAD_BF16, out


def _address(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _laid_out(scale: Tensor) -> Tensor:
    """Saved scales of a weight held by the caller, whose rows' padding hooks on saved tensors may have left out."""
    if scale.stride(0) % 4 == 0:
        return scale
    padded = torch.empty(scale.size(0), -(-scale.size(1) // 4) * 4, dtype=SCALE, device=scale.device)[:, :scale.size(1)]
    return padded.copy_(scale)


def _rows_of(x: Tensor) -> int:
    n = 1
    for d in x.shape[:-1]:
        n = n * d
    return n


def _scale_like(like: Tensor, rows: int, cols: int) -> Tensor:
    return like.new_empty((rows, -(-_blocks(cols) // 4) * 4), dtype=SCALE)


# The ops are registered by their schemas, for tracing and fake tensors, and differentiated by the functions below. A forward and
# backward of 515 x 768 x 768 from Python: 143 us; with the gradient registered 168; through torch.library.custom_op 193.
_OPS = torch.library.Library("nanochat_amd", "FRAGMENT")
_HELD = "Tensor? {0}codes, Tensor? {0}scale, Tensor? {0}codes_t, Tensor? {0}scale_t, Tensor? {0}grad"


def _op(name: str, schema: str, run, fake) -> torch._ops.OpOverload:
    _OPS.define(f"{name}{schema}")
    _OPS.impl(name, run, "CUDA")
    torch.library.register_fake(f"nanochat_amd::{name}", fake, lib=_OPS)
    return getattr(torch.ops.nanochat_amd, name).default


def _run_linear(x: Tensor, weight: Tensor, codes: Tensor | None, scale: Tensor | None, codes_t: Tensor | None,
                scale_t: Tensor | None, grad: Tensor | None) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """-> y, then what the backward reads: x's codes and scales, the weight's transposed codes and scales."""
    rows = _as_rows(x, "x", (BF16,))
    (m, k), n, device = rows.shape, weight.size(0), x.device
    if weight.dim() == 2 and k != weight.size(1):
        raise ValueError(f"x has {k} columns for a weight of {tuple(weight.shape)}")
    with device_guard(x):
        w, ws, pitch, made_t, made_ts = _held(weight, "weight", codes, scale, codes_t, scale_t, grad, device)
        x8, xs = torch.empty(m, k, dtype=CODES, device=device), _whole_scale(x, m, k)
        y = torch.empty(*x.shape[:-1], n, dtype=BF16, device=device)
        check(hip_library().nc_fp8_linear_fwd(rows.data_ptr(), rows.stride(0), w.data_ptr(), ws.data_ptr(), pitch, m, n, k,
                                              x8.data_ptr(), xs.data_ptr(), xs.size(1), y.data_ptr(), stream()))
    return y, x8, xs, made_t, made_ts


def _fake_linear(x, weight, codes, scale, codes_t, scale_t, grad):
    rows, (n, k) = _rows_of(x), weight.shape
    made = codes is None
    return (x.new_empty((*x.shape[:-1], n)), x.new_empty((rows, k), dtype=CODES), _scale_like(x, rows, k),
            x.new_empty((k, n) if made else (0,), dtype=CODES),
            _scale_like(x, _blocks(k), n) if made else x.new_empty(0, dtype=SCALE))


def _run_linear_bwd(dy: Tensor, x8: Tensor, xs: Tensor, codes_t: Tensor, scale_t: Tensor, grad: Tensor | None, need_x: bool,
                    need_w: bool, wide: bool) -> tuple[Tensor, Tensor]:
    """-> dx [rows, K], dw (either empty where it is not wanted; dw also where it was added into grad)."""
    rows, lib = _as_rows(dy, "dy", (BF16,)), hip_library()
    if need_w:
        rows = _dense(rows)
    (m, n), k = rows.shape, x8.size(-1)
    _check_kept(x8, xs, ("x8", "xs"), m, k, 1, dy.device)
    if need_x:
        _check_kept(codes_t, scale_t, ("codes_t", "scale_t"), k, n, BLOCK, dy.device)
    with device_guard(dy):
        dx = torch.empty(m, k, dtype=BF16, device=dy.device) if need_x else dy.new_empty(0)
        dw, mode, into = _layer_grad(n, k, grad, need_w, wide, dy, "grad")
        if m == 0:
            return dx, dw.zero_()
        need = lib.nc_fp8_linear_bwd_workspace_bytes(m, n, k, need_x, mode)
        ws = _workspace(dy, need)
        check(lib.nc_fp8_linear_bwd(rows.data_ptr(), rows.stride(0), x8.data_ptr(), xs.data_ptr(), xs.stride(0),
                                    codes_t.data_ptr(), scale_t.data_ptr(), scale_t.stride(0), m, n, k,
                                    dx.data_ptr() if need_x else None, _address(into), mode, ws.data_ptr(), need, stream()))
    return dx, dw


def _fake_linear_bwd(dy, x8, xs, codes_t, scale_t, grad, need_x, need_w, wide):
    k = x8.size(1)
    return (dy.new_empty((x8.size(0), k) if need_x else (0,)),
            dy.new_empty((dy.size(-1), k), dtype=F32 if wide else BF16) if need_w and grad is None else dy.new_empty(0))


_linear_bwd = _op("checkpointed_linear_bwd", "(Tensor dy, Tensor x8, Tensor xs, Tensor codes_t, Tensor scale_t, "
                  "Tensor(a!)? grad, bool need_x, bool need_w, bool wide) -> (Tensor, Tensor)", _run_linear_bwd,
                  _fake_linear_bwd)
_linear = _op("checkpointed_linear", f"(Tensor x, Tensor weight, {_HELD.format('')}) -> "
              "(Tensor, Tensor, Tensor, Tensor, Tensor)", _run_linear, _fake_linear)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx: FunctionCtx, *inputs: Tensor | None) -> Tensor:
        x, weight, codes, _, codes_t, scale_t, grad = inputs = inputs[:7]   # without _asking's
        y, x8, xs, made_t, made_ts = _linear(*inputs)
        ctx.x_shape, ctx.wide, ctx.grad = x.shape, weight.dtype == F32, grad   # grad not saved: it may change until it is added to
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x8, xs, *((codes_t, scale_t) if codes is not None else (made_t, made_ts)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: FunctionCtx, dy: Tensor | None) -> tuple:
        if dy is None:
            return (None,) * 8
        grad, need_x = ctx.grad, ctx.needs_input_grad[0]
        need_w = ctx.needs_input_grad[1] or grad is not None
        x8, xs, codes_t, scale_t = ctx.saved_tensors
        dx, dw = _linear_bwd(dy, x8, xs, codes_t, _laid_out(scale_t), grad, need_x, need_w, ctx.wide)
        return (dx.view(ctx.x_shape) if need_x else None, dw if need_w and grad is None else None, *(None,) * 6)



_NOT_HELD = (None, None, None, None)


with torch.inference_mode(False):
    _ASKS = torch.zeros((), device="cpu", requires_grad=True)   # has a call recorded whose other inputs do not; gets no gradient


def _asking(grads: tuple, inputs: tuple) -> Tensor | None:
    """The input that has a call with gradient buffers recorded where nothing else would."""
    if not torch.is_grad_enabled() or all(g is None for g in grads) or any(t.requires_grad for t in inputs):
        return None
    return _ASKS


def checkpointed_linear(x: Tensor, weight: Tensor, weight8: Fp8Weight | None = None, grad: Tensor | None = None) -> Tensor:
    """x bf16 [..., K] through a linear layer in 8-bit products, bf16 [..., N], differentiable in x and weight (bf16 or fp32
    [N, K], N and K multiples of 16 up to 65,536). Kept for the backward is x's 8-bit form alone, not x. With x8, dy8, w8 the 8-bit forms:

        y = x8 w8^T      dx = dy8 w8      dw = dy^T x8   (dy itself, fp32 sums)

    weight8: quantize_weight(weight, transpose=True), which a program that uses a weight more than once a step keeps; made in
    the call when absent. grad: None (dw is returned to autograd, in the weight's type), or an fp32 [N, K] buffer that dw is
    added to in the backward, autograd then getting none for the weight; with a buffer the call is recorded (unless under
    torch.no_grad()) and dw made whether or not x or weight requires a gradient. The gradients themselves cannot be
    differentiated."""
    return _Linear.apply(x, weight, *(weight8 or _NOT_HELD), grad, _asking((grad,), (x, weight)))


def _run_mlp(x: Tensor, fc: Tensor, proj: Tensor, fc_codes: Tensor | None, fc_scale: Tensor | None, fc_codes_t: Tensor | None,
             fc_scale_t: Tensor | None, fc_grad: Tensor | None, proj_codes: Tensor | None, proj_scale: Tensor | None,
             proj_codes_t: Tensor | None, proj_scale_t: Tensor | None, proj_grad: Tensor | None,
             fast: bool = False) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """-> y, then what the backward reads: the codes and scales of x, of the hidden activations, and of both transposes."""
    rows, device = _as_rows(x, "x", (BF16,)), x.device
    if fc.dim() == proj.dim() == 2 and (rows.size(1) != fc.size(1) or proj.size(1) != fc.size(0)):
        raise ValueError(f"x has {rows.size(1)} columns, fc is {tuple(fc.shape)}, proj {tuple(proj.shape)}")
    with device_guard(x):
        f, fs, f_pitch, f_t, f_ts = _held(fc, "fc", fc_codes, fc_scale, fc_codes_t, fc_scale_t, fc_grad, device)
        p, ps, p_pitch, p_t, p_ts = _held(proj, "proj", proj_codes, proj_scale, proj_codes_t, proj_scale_t, proj_grad, device)
        (m, c), (n, hidden) = rows.shape, proj.shape
        x8, xs = torch.empty(m, c, dtype=CODES, device=device), _whole_scale(x, m, c)
        a8, a_s = torch.empty(m, hidden, dtype=CODES, device=device), _whole_scale(x, m, hidden)
        y = torch.empty(*x.shape[:-1], n, dtype=BF16, device=device)
        call = hip_library().nc_fp8_mlp_fwd_fast if fast else hip_library().nc_fp8_mlp_fwd
        check(call(rows.data_ptr(), rows.stride(0), f.data_ptr(), fs.data_ptr(), f_pitch, p.data_ptr(), ps.data_ptr(), p_pitch, m, c,
                   hidden, n, x8.data_ptr(), xs.data_ptr(), xs.size(1), a8.data_ptr(), a_s.data_ptr(), a_s.size(1), y.data_ptr(),
                   stream()))
    return y, x8, xs, a8, a_s, f_t, f_ts, p_t, p_ts


def _fake_mlp(x, fc, proj, fc_codes, fc_scale, fc_codes_t, fc_scale_t, fc_grad, proj_codes, proj_scale, proj_codes_t,
              proj_scale_t, proj_grad, fast=False):
    rows, (hidden, k), n = _rows_of(x), fc.shape, proj.size(0)

    def kept(made, rows_t, cols_t):
        return (x.new_empty((rows_t, cols_t) if made else (0,), dtype=CODES),
                _scale_like(x, _blocks(rows_t), cols_t) if made else x.new_empty(0, dtype=SCALE))

    return (x.new_empty((*x.shape[:-1], n)), x.new_empty((rows, k), dtype=CODES), _scale_like(x, rows, k),
            x.new_empty((rows, hidden), dtype=CODES), _scale_like(x, rows, hidden), *kept(fc_codes is None, k, hidden),
            *kept(proj_codes is None, hidden, n))


def _run_mlp_bwd(dy: Tensor, x8: Tensor, xs: Tensor, a8: Tensor, a_s: Tensor, fc_codes_t: Tensor, fc_scale_t: Tensor,
                 proj_codes_t: Tensor, proj_scale_t: Tensor, fc_grad: Tensor | None, proj_grad: Tensor | None, need_x: bool,
                 need_fc: bool, need_proj: bool, fc_wide: bool, proj_wide: bool) -> tuple[Tensor, Tensor, Tensor]:
    """-> dx [rows, C], dfc, dproj (each empty where it is not wanted, or was added into its buffer)."""
    rows, lib = _as_rows(dy, "dy", (BF16,)), hip_library()
    if need_proj:
        rows = _dense(rows)
    (m, n), c, hidden = rows.shape, x8.size(-1), a8.size(-1)
    _check_kept(x8, xs, ("x8", "xs"), m, c, 1, dy.device)
    _check_kept(a8, a_s, ("a8", "a_s"), m, hidden, 1, dy.device)
    if need_x:
        _check_kept(fc_codes_t, fc_scale_t, ("fc_codes_t", "fc_scale_t"), c, hidden, BLOCK, dy.device)
    if need_x or need_fc:
        _check_kept(proj_codes_t, proj_scale_t, ("proj_codes_t", "proj_scale_t"), hidden, n, BLOCK, dy.device)
    with device_guard(dy):
        dx = torch.empty(m, c, dtype=BF16, device=dy.device) if need_x else dy.new_empty(0)
        dfc, fc_mode, fc_into = _layer_grad(hidden, c, fc_grad, need_fc, fc_wide, dy, "fc_grad")
        dproj, proj_mode, proj_into = _layer_grad(n, hidden, proj_grad, need_proj, proj_wide, dy, "proj_grad")
        if m == 0:
            return dx, dfc.zero_(), dproj.zero_()
        need = lib.nc_fp8_mlp_bwd_workspace_bytes(m, c, hidden, n, need_x, fc_mode, proj_mode)
        ws = _workspace(dy, need)
        check(lib.nc_fp8_mlp_bwd(
            rows.data_ptr(), rows.stride(0), x8.data_ptr(), xs.data_ptr(), xs.stride(0), a8.data_ptr(), a_s.data_ptr(),
            a_s.stride(0), fc_codes_t.data_ptr(), fc_scale_t.data_ptr(), fc_scale_t.stride(0), proj_codes_t.data_ptr(),
            proj_scale_t.data_ptr(), proj_scale_t.stride(0), m, c, hidden, n, dx.data_ptr() if need_x else None,
            _address(fc_into), fc_mode, _address(proj_into), proj_mode, ws.data_ptr(), need, stream()))
    return dx, dfc, dproj


def _fake_mlp_bwd(dy, x8, xs, a8, a_s, fc_codes_t, fc_scale_t, proj_codes_t, proj_scale_t, fc_grad, proj_grad, need_x, need_fc,
                  need_proj, fc_wide, proj_wide):
    (rows, k), hidden, n = x8.shape, a8.size(1), dy.size(-1)
    return (dy.new_empty((rows, k) if need_x else (0,)),
            dy.new_empty((hidden, k), dtype=F32 if fc_wide else BF16) if need_fc and fc_grad is None else dy.new_empty(0),
            dy.new_empty((n, hidden), dtype=F32 if proj_wide else BF16) if need_proj and proj_grad is None else dy.new_empty(0))


_mlp_bwd = _op("checkpointed_mlp_bwd", "(Tensor dy, Tensor x8, Tensor xs, Tensor a8, Tensor a_s, Tensor fc_codes_t, "
               "Tensor fc_scale_t, Tensor proj_codes_t, Tensor proj_scale_t, Tensor(a!)? fc_grad, Tensor(b!)? proj_grad, "
               "bool need_x, bool need_fc, bool need_proj, bool fc_wide, bool proj_wide) -> (Tensor, Tensor, Tensor)",
               _run_mlp_bwd, _fake_mlp_bwd)
_mlp = _op("checkpointed_mlp", f"(Tensor x, Tensor fc, Tensor proj, {_HELD.format('fc_')}, {_HELD.format('proj_')}, "
           f"bool fast=False) -> ({', '.join(['Tensor'] * 9)})", _run_mlp, _fake_mlp)


class _Mlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx: FunctionCtx, *inputs: Tensor | bool | None) -> Tensor:
        x, fc, proj = inputs[:3]
        f, p = inputs[3:8], inputs[8:13]
        y, x8, xs, a8, a_s, f_t, f_ts, p_t, p_ts = _mlp(*inputs[:14])   # without _asking's
        ctx.x_shape, ctx.fc_wide, ctx.proj_wide = x.shape, fc.dtype == F32, proj.dtype == F32
        ctx.fc_grad, ctx.proj_grad = f[4], p[4]
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x8, xs, a8, a_s, *(f[2:4] if f[0] is not None else (f_t, f_ts)),
                              *(p[2:4] if p[0] is not None else (p_t, p_ts)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: FunctionCtx, dy: Tensor | None) -> tuple:
        if dy is None:
            return (None,) * 15
        fc_grad, proj_grad, need_x = ctx.fc_grad, ctx.proj_grad, ctx.needs_input_grad[0]
        need_fc, need_proj = ctx.needs_input_grad[1] or fc_grad is not None, ctx.needs_input_grad[2] or proj_grad is not None
        x8, xs, a8, a_s, f_t, f_ts, p_t, p_ts = ctx.saved_tensors
        dx, dfc, dproj = _mlp_bwd(dy, x8, xs, a8, a_s, f_t, _laid_out(f_ts), p_t, _laid_out(p_ts), fc_grad, proj_grad, need_x,
                                  need_fc, need_proj, ctx.fc_wide, ctx.proj_wide)
        return (dx.view(ctx.x_shape) if need_x else None, dfc if need_fc and fc_grad is None else None,
                dproj if need_proj and proj_grad is None else None, *(None,) * 12)



def checkpointed_mlp(x: Tensor, fc: Tensor, proj: Tensor, fc8: Fp8Weight | None = None, proj8: Fp8Weight | None = None,
                     fc_grad: Tensor | None = None, proj_grad: Tensor | None = None, fast: bool = False) -> Tensor:
    """x bf16 [..., C] through proj(relu(fc(x))^2) in 8-bit products, bf16 [..., N], differentiable in x, fc [F, C] and proj
    [N, F] (bf16 or fp32, all sizes multiples of 16 up to 65,536). Kept for the backward are the 8-bit forms of x and of the squared
    activations a, C + F bytes a token where bf16 keeps x, the sums before the square and the squares in 2 C + 4 F. With x8
    and so on the 8-bit forms, f8 and p8 the weights':

        a = relu(x8 f8^T)^2      y = a8 p8^T      dh = bf16((dy8 p8) 2 sqrt(a8))
        dx = dh8 f8      dfc = dh^T x8      dproj = dy^T a8

    The derivative of the square is read from the checkpoint itself: 2 relu(h) = 2 sqrt(a). fc8, proj8, fc_grad and proj_grad
    as checkpointed_linear's weight8 and grad. fast: as fp8_mlp's, of x8 f8^T; what it says of the result holds for dproj, too."""
    return _Mlp.apply(x, fc, proj, *(fc8 or _NOT_HELD), fc_grad, *(proj8 or _NOT_HELD), proj_grad, fast,
                      _asking((fc_grad, proj_grad), (x, fc, proj)))
