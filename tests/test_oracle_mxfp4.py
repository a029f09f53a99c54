"""The numpy oracles of MXFP4 and of the 8-bit moments (CPU only)."""

import numpy as np
import pytest

from oracle import adamw as oadam
from oracle import mxfp4 as omx


def test_known_blocks():
    x = np.zeros(32)
    x[:10] = [6, -6, 5, 2.5, 1.75, 0.25, 0.75, 3.5, -0.0, 7]
    codes, scales = omx.quantize(x)
    # amax 7 = 2^2 * 1.75: scale 2^0; 7 saturates; ties go to the even code.
    assert scales[0] == 127
    got = omx.dequantize(codes, scales, 32)[:10]
    assert got.tolist() == [6, -6, 4, 2, 2, 0, 1, 4, 0, 6]
    assert np.signbit(got[8])
    # Element 2 i in the low nibble.
    assert codes[0] == 7 | (15 << 4)


@pytest.mark.parametrize("amax,scale", [(0.0, 0), (2.0 ** -149, 0), (2.0 ** -125, 0), (2.0 ** -124, 1),
                                        (1.0, 125), (7.99, 127), (8.0, 128), (3.4e38, 252)])
def test_scale_bytes(amax, scale):
    assert omx.quantize(np.full(32, amax))[1][0] == scale


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_bad_value_poisons_its_block_only(bad):
    x = np.ones(64)
    x[40] = bad
    codes, scales = omx.quantize(x)
    assert scales.tolist() == [125, 255]
    assert not codes[16:].any()
    assert np.isnan(omx.dequantize(codes, scales, 64)[32:]).all()


def test_rounding_is_at_most_half_a_spacing():
    x = np.random.default_rng(0).normal(size=(64, 96))
    codes, scales = omx.quantize(x)
    q = omx.dequantize(codes, scales, 96)
    s = np.repeat(2.0 ** (scales.astype(float) - 127), 32, axis=-1)
    y = np.abs(x) / s
    spacing = np.where(y < 2, 0.5, np.where(y < 4, 1.0, 2.0))
    inside = y <= 6
    assert (np.abs(x - q)[inside] <= (spacing * s / 2)[inside]).all()
    assert (np.abs(q)[~inside] == 6 * s[~inside]).all()


def test_ragged_rows_are_padded_with_zeros():
    codes, scales = omx.quantize(np.ones((3, 33)))
    assert codes.shape == (3, 32) and scales.shape == (3, 2)
    assert codes[0, 16] & 15 == 6 and not codes[0, 17:].any() and codes[0, 16] >> 4 == 0


@pytest.mark.parametrize("ebits,signed", [(4, True), (5, False)])
def test_moment_codes_are_fixed_points(ebits, signed):
    levels = oadam.level_table(ebits)
    assert (np.diff(levels) > 0).all() and levels[-1] == 1.875
    x = levels.astype(np.float32)
    x = np.concatenate([x, -x]) if signed else x
    n = x.size
    # With 1.875 in each block the exponent is 0 and every level its own code.
    x = np.concatenate([np.concatenate([x[i:i + 127], [1.875]]) for i in range(0, n, 127)]).astype(np.float32)
    for bits in (0, 65535):
        codes, exps = oadam.encode(x, ebits, signed, np.full(x.size, bits))
        # (the last block may be short of 128 values, all hold a 1.875)
        assert (exps == 127).all()
        assert np.array_equal(oadam.decode(codes, exps, ebits, signed), x)


def test_stochastic_rounding_is_unbiased():
    rng = np.random.default_rng(1)
    x = np.abs(rng.normal(size=128)).astype(np.float32)
    total = np.zeros(128)
    steps = 4000
    for t in range(steps):
        low, _ = oadam.noise(128, 7, t, 0)
        total += oadam.decode(*oadam.encode(x, 4, True, low), 4, True)
    spacing = np.ldexp(1.0, np.frexp(x)[1] - 1 - 3)
    # The mean of `steps` roundings, each off by less than a spacing: within 5 standard
    # errors of at most spacing / 2 / sqrt(steps).
    assert (np.abs(total / steps - x) <= 5 * spacing / 2 / np.sqrt(steps)).all()


def test_noise_differs_by_seed_step_group_and_position():
    base = oadam.noise(4096, 1, 2, 3)[0]
    for other in (oadam.noise(4096, 2, 2, 3), oadam.noise(4096, 1, 3, 3), oadam.noise(4096, 1, 2, 4),
                  oadam.noise(4096, 1, 2, 3, at=4096)):
        assert (base != other[0]).mean() > 0.99
