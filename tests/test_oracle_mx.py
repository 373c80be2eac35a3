"""CPU: the NumPy statement of microscaled 4-bit rows against values worked out by hand and the format's properties."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import mx


def test_a_block_by_hand():
    x = np.zeros((1, 32))
    # Largest 7.9: floor(log2) = 2, scale 2^0; above 6 is 6.  Ties go to the even index.
    x[0, :16] = [7.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.26, -0.0, 5.01, -5.0, 6.9, 0.7499, 3.4999, 1e-30]
    codes, scales = mx.quantize(x)
    assert scales.tolist() == [[127]]
    n = np.stack([codes & 15, codes >> 4], -1).reshape(-1)
    assert n[:16].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 9, 8, 7, 14, 7, 1, 5, 0]
    assert mx.dequantize(codes, scales)[0, :8].tolist() == [6, 0, 1, 1, 2, 2, 4, 4]


def test_scales_of_powers_of_two_and_their_ends():
    for e in (-149, -130, -126, -125, -124, -1, 0, 1, 100, 127):
        x = np.full((1, 32), np.ldexp(1.0, e))
        codes, scales = mx.quantize(x)
        assert scales[0, 0] == max(e - 2, -127) + 127
        v = mx.dequantize(codes, scales)
        if e >= -128:  # below, 2^e is less than half of 2^-127 times 0.5, or a tie that goes to zero
            assert (v == x).all()


def test_bad_blocks_padding_and_zeros():
    x = np.ones((2, 70))
    x[0, 40], x[1, 3] = np.nan, -np.inf
    codes, scales = mx.quantize(x)
    assert codes.shape == (2, 48) and scales.shape == (2, 3)
    assert scales[0, 1] == 255 and scales[1, 0] == 255 and not codes[0, 16:32].any() and not codes[1, :16].any()
    assert np.isnan(mx.dequantize(codes, scales)[0, 32:64]).all()
    assert not codes[0, 35:].any()  # columns 70.. of the last block
    codes, scales = mx.quantize(np.zeros((1, 32)))
    assert not codes.any() and not scales.any()


@pytest.mark.parametrize("seed", [0, 1])
def test_nearest_level(seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((64, 96)) * np.exp2(rng.integers(-20, 20, (64, 1)))
    codes, scales = mx.quantize(x)
    v = mx.dequantize(codes, scales)
    s = np.repeat(np.exp2(scales.astype(float) - 127), 32, axis=1)
    gap = np.where(np.abs(v) < 2 * s, 0.25, np.where(np.abs(v) < 4 * s, 0.5, 1.0)) * s  # half the step above a level
    assert (np.abs(x - v)[np.abs(x) <= 6 * s] <= gap[np.abs(x) <= 6 * s]).all()
    assert (np.abs(x) < 8 * s).all()
