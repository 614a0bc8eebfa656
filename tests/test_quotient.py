"""The quantisers' quotient by the constant 448 (corrected_quotient in rows.cuh), in whole numbers: a product with the rounded reciprocal and
one correction by the exact remainder give the correctly rounded quotient for every significand."""
import numpy as np


def nearest_even(num, shift):
    """round(num / 2^shift), ties to even"""
    low, half, q = num & ((1 << shift) - 1), 1 << (shift - 1), num >> shift
    return q + ((low > half) | ((low == half) & (q & 1 == 1)))


def test_scales_are_correctly_rounded_for_every_significand():
    m = np.arange(1 << 23, 1 << 24, dtype=np.int64)  # v, a float's significand as a whole number
    R = round(2 ** 32 / 448)  # r = R 2^-32
    assert 1 << 23 <= R < 1 << 24 and np.float32(1) / np.float32(448) == np.float32(R) * np.float32(2.0 ** -32)
    # the quotient lies in (2^14, 2^16): units in the last place of 2^-9 and 2^-8
    def to_float(num, bits):
        """num 2^-bits as a float, in units of 2^-9"""
        fine = nearest_even(num, bits - 9)
        return np.where(num >> bits < 1 << 15, fine, 2 * nearest_even(num, bits - 8))

    q = to_float(m * R, 32)
    rem = (m << 9) - q * 448  # in units of 2^-9
    assert np.abs(rem).max() < 1 << 24  # exact as a float
    got = to_float((q << 32) + rem * R, 41)
    unit = np.where(m < 448 << 15, 1, 2)  # of the true quotient, in 2^-9
    num, den = m << 9, 448 * unit
    whole, left = num // den, num % den
    want = (whole + ((2 * left > den) | ((2 * left == den) & (whole & 1 == 1)))) * unit
    assert (got == want).all()
    # the same by the host's division, which is IEEE's
    v = m.astype(np.float32)
    assert (v / np.float32(448) == got.astype(np.float64) * 2.0 ** -9).all()
