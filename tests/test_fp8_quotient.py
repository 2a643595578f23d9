"""The quotient whose code a value gets (csrc/fp8_common.h): q = fma(-fma(near, s, -v), inverse, near) with near = v inverse and
inverse = 1 / s, each rounded to fp32.  It has the code of v / s rounded to fp32, for every v and s (CPU only).

q is off by at most 2^-22 units of its last place before it is rounded: near by 1.5 units, its remainder by 2^-24 of it for its own rounding,
and 2^-24 for that of the inverse.  So q is another value than the quotient's only if that is within 2^-22 units of the middle of
two fp32 values, and its code another only if one of the two is a tie of codes, an odd multiple of 2^-4 of a power of two (of a
coarser one below the normal codes).  Here are all fractions of s, all ties and both middles next to each, to twice that distance."""

from __future__ import annotations

from fractions import Fraction

import numpy as np

# a tie in 32nds, with the leading one at 16: T / 16 for odd T from 17 on, and odd T below, shifted up
TIES = sorted({t << (5 - t.bit_length()) for t in range(1, 32, 2)})


def rounded(x):
    """To 24 bits, ties to even; no end of range."""
    if x == 0:
        return x
    size = abs(x)
    power = size.numerator.bit_length() - size.denominator.bit_length()
    if Fraction(2) ** power > size:
        power -= 1
    unit = Fraction(2) ** (power - 23)
    return (1 if x > 0 else -1) * round(size / unit) * unit  # (round: to even)


def quotient(v, s):
    inverse = rounded(1 / s)
    near = rounded(v * inverse)
    return rounded(near - rounded(near * s - v) * inverse)


def test_rounding():
    rng = np.random.default_rng(0)
    for x in np.exp(rng.uniform(-20, 20, 200)) * rng.choice([-1, 1], 200):
        assert float(rounded(Fraction(float(x)))) == float(np.float32(x))
    assert rounded(Fraction((1 << 24) + 1)) == 1 << 24 and rounded(Fraction((1 << 24) + 3)) == (1 << 24) + 4


def test_quotients_next_to_middles_beside_ties():
    s = np.arange(1 << 23, 1 << 24, dtype=np.int64)
    found = 0
    for tie in TIES:
        at = tie << 19                                              # in units of 2^-23, from 1 to 2
        for middle in (4 * at + 2, 4 * at - (1 if tie == 16 else 2)):  # of 2^-25; below a power of two values are half as far apart
            exact = middle * s                                      # of 2^-25 of s's last place: below 2^51
            for shift in (25, 26):                                  # v of s's power of two, and of the next
                v = (exact + (1 << (shift - 1))) >> shift
                off = exact - (v << shift)
                fits = (v >= 1 << 23) & (v < 1 << 24)
                assert not (fits & (off == 0)).any()                # no quotient is in the middle of two values
                # (a unit of the quotient's last place is 4 s of these)
                for i in np.nonzero(fits & (np.abs(off) < 2.0 ** -21 * 4 * s))[0]:
                    x, y = Fraction(int(v[i]) << (shift - 25)), Fraction(int(s[i]))
                    assert quotient(x, y) == rounded(x / y), (x, y)
                    found += 1
    assert found > 100


def test_random_quotients():
    rng = np.random.default_rng(1)
    for v, s in rng.integers(1 << 23, 1 << 24, (3000, 2)):
        x, y = Fraction(int(v)), Fraction(int(s))
        assert abs(quotient(x, y) - rounded(x / y)) <= Fraction(1, 1 << 23)
        assert quotient(-x, y) == -quotient(x, y)
