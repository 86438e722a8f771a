"""Cosines and sines of position times frequency, with the angle in whole numbers throughout.

A 64-bit product of a far position and a frequency has lost the very turns that a rotation is about, so
it is no oracle there. There is no counterpart in the reference.
"""

from __future__ import annotations

import math

import numpy as np

BITS = 512  # of 1 / (2 pi), for |position * frequency| below 2^400


def _inverse_turn() -> int:
    """2^BITS / (2 pi), pi by Machin's formula."""

    one = 1 << (BITS + 64)

    def atan_of_inverse(n: int) -> int:
        term, total, odd, sign = one // n, 0, 1, 1
        while term:
            total += sign * (term // odd)
            term, odd, sign = term // (n * n), odd + 2, -sign
        return total

    pi = 4 * (4 * atan_of_inverse(5) - atan_of_inverse(239))
    return (one << BITS) // (2 * pi)


_INVERSE = _inverse_turn()


def cos_sin(positions: np.ndarray, frequencies: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """float64 [positions, frequencies] each: of whole positions and any finite frequencies, to 2^-50."""

    cos = np.empty((len(positions), len(frequencies)))
    sin = np.empty_like(cos)
    for j, f in enumerate(frequencies):
        n, d = float(f).as_integer_ratio()
        one = d << BITS
        for i, p in enumerate(positions):
            x = int(p) * n * _INVERSE % one  # of a turn
            eighth, rest = divmod(8 * x + one // 2, one)  # the nearest one, so that what is left is small
            a = 2.0 * math.pi * ((rest - one // 2) / (8 * one))
            c, s = math.cos(a), math.sin(a)
            h = math.sqrt(0.5)
            u, v = ((1.0, 0.0), (h, h), (0.0, 1.0), (-h, h), (-1.0, 0.0), (-h, -h), (0.0, -1.0), (h, -h))[eighth % 8]
            cos[i, j], sin[i, j] = c * u - s * v, s * u + c * v
    return cos, sin
