"""Plain 64-bit forms of the norm and the 8-bit operators (numpy), and what their results may differ by, for the tests."""

from __future__ import annotations

import numpy as np

BLOCK = 128
HALF_STEP = {"float16": 2.0 ** -11, "float32": 2.0 ** -24}   # of a rounding, relative
HALF_LEAST = {"float16": 2.0 ** -25, "float32": 2.0 ** -150}  # below the normal values
# A norm in fp32: its sum of positive squares goes through at most 32 + 6 + 16 additions and two roundings before
# them, half of which the root takes over; the root, the products and h add four more.
NORM_OFF = 40 * 2.0 ** -24


def blocks_of(n):
    return -(-n // BLOCK)


def value(codes):
    """e4m3: sign, four bits of exponent (bias 7), three of fraction."""
    table = np.zeros(256)
    for code in range(256):
        exponent, fraction = (code >> 3) & 15, code & 7
        size = fraction * 2.0 ** -9 if exponent == 0 else (1 + fraction / 8) * 2.0 ** (exponent - 7)
        table[code] = np.nan if code & 127 == 127 else -size if code & 128 else size
    return table[codes]


def spread(scales, width):
    """Scales [blocks, rows] as [rows, width]."""
    return np.repeat(scales.T.astype(np.float64), BLOCK, axis=1)[:, :width]


def norm(x, residual, weight, eps):
    """(y, h) in 64 bits."""
    h = x.astype(np.float64)
    if residual is not None:
        h = h + residual.astype(np.float64)
    with np.errstate(all="ignore"):
        top = np.max(np.abs(h), axis=1, keepdims=True)
        top = np.where((top > 0) & np.isfinite(top), top, 1.0)
        root = top * np.sqrt(np.mean((h / top) ** 2, axis=1, keepdims=True) + eps / top ** 2)
        return h / root * weight.astype(np.float64), h


def gated(x):
    half = x.shape[1] // 2
    g, u = x[:, :half].astype(np.float64), x[:, half:].astype(np.float64)
    with np.errstate(all="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def check_rounded(got, want, dtype, off=0.0):
    """One rounding to dtype of values that are off by at most `off` of them; what is not finite is the same."""
    assert got.dtype == dtype
    with np.errstate(all="ignore"):
        limit = np.finfo(dtype).max * (1 + HALF_STEP[dtype])
        want = np.where(np.abs(want) >= limit, np.sign(want) * np.inf, want)
    sure = ~(np.abs(want) > 0.999 * np.finfo(dtype).max)  # next to the border either is right
    assert np.array_equal(np.isnan(got), np.isnan(want))
    got64 = got.astype(np.float64)
    fine = np.isfinite(want) & sure
    assert np.array_equal(got64[~fine & ~np.isnan(want) & sure], want[~fine & ~np.isnan(want) & sure])
    error = np.abs(got64 - np.where(fine, want, 0))[fine]
    bound = np.abs(want)[fine] * (HALF_STEP[dtype] + off) + HALF_LEAST[dtype]
    assert (error <= bound).all(), float((error / bound).max())


def check_codes(codes, scales, want, off):
    """Codes and scales of values that are off by at most `off` of them: a scale is its block's largest finite magnitude
    / 448, 2^-126 at least; a code is the nearest value, off by half a step (2^-4 of it, 2^-10 below the normal ones)."""
    rows, width = want.shape
    assert codes.shape == (rows, width) and scales.shape == (blocks_of(width), rows)
    finite = np.isfinite(want)
    size = np.where(finite, np.abs(want), 0.0)
    for b in range(blocks_of(width)):
        top = np.maximum(size[:, b * BLOCK:(b + 1) * BLOCK].max(axis=1) / 448.0, 2.0 ** -126)
        assert (np.abs(scales[b] - top) <= (off + 2.0 ** -22) * top + 2.0 ** -149).all(), b
    assert np.array_equal(np.isnan(value(codes)), ~finite)
    s = spread(scales, width)
    got = np.where(finite, value(codes), 0.0)
    u = np.where(finite, want, 0.0) / s
    error = np.abs(got - u)
    # the quotient is rounded twice (1 / s, and its product), and the value it is of is off; 448 is the largest code
    bound = np.maximum(np.abs(u) * 2.0 ** -4, 2.0 ** -10) + np.abs(u) * (off + 2.0 ** -22)
    assert (error <= bound).all(), float((error / bound).max())


def random_codes(rng, shape):
    """Codes of all sizes, none of them NaN."""
    codes = rng.integers(0, 256, shape).astype(np.uint8)
    codes[codes & 127 == 127] = 0x7E
    return codes


def linear(x, x_scales, w, w_scales):
    """(out, the sum of its terms' magnitudes) in 64 bits."""
    xs, ws = _scaled(x, x_scales, w, w_scales)
    return xs @ ws.T, np.abs(xs) @ np.abs(ws).T


def _scaled(x, x_scales, w, w_scales):
    n, k = w.shape
    return (value(x) * spread(x_scales, k),
            value(w) * np.repeat(np.repeat(w_scales.astype(np.float64), BLOCK, 0)[:n], BLOCK, 1)[:, :k])


def _power(values):
    """The power of two that a code's exponent gives: 2^-6 for those below the normal values, 0 for zero."""
    size = np.where(np.isfinite(values), np.abs(values), 0.0)
    return np.where(size > 0, np.exp2(np.floor(np.log2(np.maximum(size, 2.0 ** -6)))), 0.0)


def cut_off(x, x_scales, w, w_scales):
    """What the 8-bit matrix instructions may cut off: within each 8 columns next to each other, a product is cut off at
    2^-13 of the largest power of two that a product's two exponents add up to.  Products there have six bits of fraction
    and lose nothing, so up to seven products lose less than 2^-13 of that power each."""
    k = x.shape[1]
    px = _power(value(x)) * spread(x_scales, k)
    pw = _power(value(w)) * np.repeat(np.repeat(w_scales.astype(np.float64), BLOCK, 0)[:w.shape[0]], BLOCK, 1)[:, :k]
    px, pw = np.nan_to_num(px), np.nan_to_num(pw)
    result = np.empty((x.shape[0], w.shape[0]))
    for row in range(x.shape[0]):
        result[row] = 7 * 2.0 ** -13 * (pw * px[row]).reshape(w.shape[0], -1, 8).max(axis=2).sum(axis=1)
    return result


def check_linear(got, want, size, k, cut=0.0):
    """One rounding to the output's type; before it a block's 128 products, exact in fp32, are added up and the blocks'
    sums scaled and added, each step off by at most 2^-23 of the terms' magnitudes (twice a rounding's half step, since
    the matrix cores may cut off bits that they align away); and what the 8-bit instructions cut off."""
    dtype = str(got.dtype)
    bound = np.abs(want) * HALF_STEP[dtype] + HALF_LEAST[dtype] + size * (BLOCK + blocks_of(k) + 4) * 2.0 ** -23 + cut * (1 + HALF_STEP[dtype])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    if dtype == "float16":
        fine &= np.abs(want) + bound < 65504
    error = np.abs(got.astype(np.float64) - want)[fine]
    assert (error <= bound[fine]).all(), float((error / bound[fine]).max())
