"""The 8-bit form of matrices and what is computed from it, in float64 — test infrastructure only.

A block of x (128 columns of a row; 128 x 128 of a weight) has the scale s = 2^e, the least with max |x| <= 448 s, e >= -126
(s = 1 for zeros), and the values rne(x / s) s, rne rounding to e4m3fn's nearest value, ties to even. A block with an infinity
or a NaN is NaN. No counterpart in the reference, whose linear layers are bf16 (model/ops/linear.py:51-57, 135-144)."""
import numpy as np

BLOCK = 128
FP8_MAX = 448.0


def exponents(amax):
    """The scale's exponent for each amax (finite float64)."""
    mantissa, e = np.frexp(np.asarray(amax, dtype=np.float64))     # amax = mantissa 2^e, mantissa in [0.5, 1)
    e = e - 9 + (mantissa > FP8_MAX / 512)
    return np.where(np.asarray(amax) > 0, np.maximum(e, -126), 0)


def e4m3_round(y):
    """Finite y, |y| <= 448, to the nearest e4m3fn value: steps of 2^(floor(log2 |y|) - 3), 2^-9 below 2^-6."""
    y = np.asarray(y, dtype=np.float64)
    size = np.maximum(np.frexp(y)[1] - 1, -6)
    step = np.ldexp(1.0, size - 3)
    return np.rint(y / step) * step


def quantize(x, rows):
    """x [R, C] float64 -> (values of the codes [R, C], exponents int [ceil(R / rows), ceil(C / 128)]); NaN blocks: NaN codes,
    exponent 128."""
    x = np.asarray(x, dtype=np.float64)
    codes, exps = np.empty_like(x), np.empty((-(-x.shape[0] // rows), -(-x.shape[1] // BLOCK)), dtype=np.int64)
    for i in range(exps.shape[0]):
        for j in range(exps.shape[1]):
            at = np.s_[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK]
            amax = np.abs(x[at]).max()
            if not np.isfinite(amax):
                exps[i, j], codes[at] = 128, np.nan
                continue
            exps[i, j] = exponents(amax)
            codes[at] = e4m3_round(np.ldexp(x[at], -exps[i, j]))
    return codes, exps


def values(codes, exps, rows):
    """What codes stand for."""
    e = np.repeat(np.repeat(exps, rows, 0), BLOCK, 1)[:codes.shape[0], :codes.shape[1]]
    return np.ldexp(np.asarray(codes, dtype=np.float64), e)


def through(x, rows):
    return values(*quantize(x, rows), rows)
