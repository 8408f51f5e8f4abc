"""Rotated positions from the definition: angles from whole-number phases, products in 64 bits."""

import numpy as np


def angles(rates, positions):
    """Angle of every (position, pair): position * rate / 2^64 of a turn, the product exact."""
    with np.errstate(over="ignore"):
        phase = positions.astype(np.int64).astype(np.uint64)[..., None] * rates.astype(np.uint64)
    return phase.astype(np.float64) * (2 * np.pi / 2.0 ** 64)


def places(rot, interleaved):
    """The elements of each pair."""
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def rotate(x, rates, positions, gain=1.0, interleaved=False, inverse=False):
    """(x [..., heads, d] float64 rotated, what its rotated elements' 32-bit error is bounded by).

    The kernels' cosines and sines are off by 2^-22: a remainder of an eighth of a turn at most,
    rounded three times (conversion, constant, product: 2.5 * 2^-24 of it, under 1.2e-7), and the
    roundings of a polynomial's last steps (2^-25 and less).  The gain, two products and a sum add at
    most 4 * 2^-24 of the pair's elements: under 2^-21 of them together."""
    a = angles(rates, positions)[..., None, :]
    c, s = gain * np.cos(a), gain * np.sin(a) * (-1 if inverse else 1)
    lo, hi = places(2 * len(rates), interleaved)
    y, bound = x.copy(), np.zeros_like(x)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    bound[..., lo] = bound[..., hi] = abs(gain) * 2.0 ** -21 * (np.abs(x[..., lo]) + np.abs(x[..., hi]))
    return y, bound
