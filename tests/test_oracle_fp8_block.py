"""The 8-bit form's oracle against torch's casts and the properties that define it."""
import numpy as np
import pytest
import torch

from oracle import fp8_block as fb


def test_rounding_is_torchs_cast():
    y = np.concatenate([np.linspace(-448, 448, 20001), np.ldexp(np.linspace(-2, 2, 4001), -6), np.ldexp(1.0, -np.arange(20))])
    y = y.astype(np.float32)
    assert np.array_equal(fb.e4m3_round(y), torch.from_numpy(y).to(torch.float8_e4m3fn).double().numpy())


def test_scale_is_the_least_power_that_holds_the_block():
    rng = np.random.default_rng(0)
    amax = np.concatenate([np.ldexp(rng.uniform(1, 2, 500), rng.integers(-110, 127, 500)), np.ldexp(1.75, np.arange(-100, 100)),
                           np.nextafter(np.ldexp(1.75, np.arange(-100, 100)), np.inf)])
    e = fb.exponents(amax)
    assert np.all(amax <= np.ldexp(448.0, e)) and np.all(amax > np.ldexp(448.0, e - 1))
    assert fb.exponents(0.0) == 0 and fb.exponents(2.0 ** -149) == -126


@pytest.mark.parametrize("rows,shape", [(1, (3, 300)), (128, (200, 400))])
def test_error_is_half_a_step(rows, shape):
    x = np.random.default_rng(1).standard_normal(shape) * np.exp2(np.random.default_rng(2).integers(-12, 12, shape))
    codes, exps = fb.quantize(x, rows)
    s = np.repeat(np.repeat(np.ldexp(1.0, exps), rows, 0), 128, 1)[:shape[0], :shape[1]]
    assert np.all(np.abs(fb.values(codes, exps, rows) - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s))
    assert np.abs(codes).max() <= 448


def test_blocks_with_an_infinity_are_nan():
    x = np.ones((2, 256))
    x[0, 3], x[1, 200] = np.inf, np.nan
    codes, exps = fb.quantize(x, 1)
    assert np.isnan(codes[0, :128]).all() and np.isnan(codes[1, 128:]).all()
    assert not np.isnan(codes[0, 128:]).any() and exps.tolist() == [[128, -8], [-8, 128]]
