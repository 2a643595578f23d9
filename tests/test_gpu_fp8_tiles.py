"""Every tile kernel of the 8-bit linear, over whole and short last steps of K, few steps and its main loop, and several tiles
(tests/fp8_tiles.py), against 64-bit sums."""

from __future__ import annotations

import numpy as np
import pytest

from tests import fp8_cases as plain, fp8_tiles
from tests.test_gpu_fp8 import operands, run_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", fp8_tiles.CASES, ids=str)
def test_whole_numbers_are_exact(hip_device, case):
    """Every result: sums of whole multiples of 2^-6 below 2^17, which fp32 holds on the way in any order (here too), and of which
    the 8-bit instructions cut nothing off (products of 1 to 9 are whole multiples of 2^(2 - 13))."""
    dtype, _, (m, n, k) = case
    print(f"[case] linear {case}", flush=True)
    rng = np.random.default_rng(m + n + k)
    codes, values = np.array([0x00, 0x38, 0x40, 0x44, 0xB8, 0xC0, 0xC4], np.uint8), np.array([0, 1, 2, 3, -1, -2, -3], np.float32)
    x, w = rng.integers(0, 7, (m, k)), rng.integers(0, 7, (n, k))
    x_scales = np.exp2(rng.integers(-3, 1, (plain.blocks_of(k), m))).astype(np.float32)
    w_scales = np.exp2(rng.integers(-3, 1, (plain.blocks_of(n), plain.blocks_of(k)))).astype(np.float32)
    assert 9 * k < 1 << 17
    xs = values[x] * np.repeat(x_scales.T, 128, axis=1)[:, :k]
    ws = values[w] * np.repeat(np.repeat(w_scales, 128, 0)[:n], 128, 1)[:, :k]
    want = xs @ ws.T
    assert want.dtype == np.float32
    got = run_linear(hip_device, codes[x], x_scales, codes[w], w_scales, dtype)
    with np.errstate(over="ignore"):
        assert np.array_equal(got, want.astype(dtype))


@pytest.mark.parametrize("case", fp8_tiles.LONG, ids=str)
def test_codes_of_all_sizes_and_such_as_are_not_numbers(hip_device, case):
    """A NaN of x is in its row, one of w in its column, and nowhere else; other results are within what their arithmetic leaves.
    (In the last tiles, whose other rows are past the end, and in the last columns.)"""
    dtype, _, (m, n, k) = case
    print(f"[case] linear {case}", flush=True)
    x, x_scales, w, w_scales = operands(m + n + k, m, n, k)
    x[m - 2, k - 1], w[n - 3, k - 2], w[1, 0] = 0x7F, 0xFF, 0x7F
    got = run_linear(hip_device, x, x_scales, w, w_scales, dtype)
    want = np.zeros((m, n), bool)
    want[m - 2], want[:, [1, n - 3]] = True, True
    assert np.array_equal(np.isnan(got), want)
    rows = np.unique(np.concatenate([[0, m // 2, m - 2, m - 1], np.random.default_rng(1).integers(0, m, 2)]))
    call = (x[rows], np.ascontiguousarray(x_scales[:, rows]), w, w_scales)
    sums, size = plain.linear(*call)
    cut = plain.cut_off(*call) if dtype == "float16" else 0.0
    plain.check_linear(got[rows], sums, np.nan_to_num(size), k, cut)
