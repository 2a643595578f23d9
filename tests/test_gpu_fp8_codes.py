"""Codes of the 8-bit operators bit for bit: those of the fp32 quotient value / scale, rounded to the nearest code, ties to the even
one, whatever the scale."""

from __future__ import annotations

import numpy as np
import pytest

from tensor_amd.kernels import fp8
from tests import fp8_cases as plain
from tests.test_gpu_fp8 import run_norm, run_quantize

pytestmark = pytest.mark.gpu

VALUES = plain.value(np.arange(127))                 # 0 to 448
TIES = (VALUES[1:] + VALUES[:-1]) / 2                # 126 of them


def want_codes(x):
    """(codes, scales) of rows of whole blocks in fp32: one division each, rounded once."""
    rows, width = x.shape
    blocks = x.astype(np.float32).reshape(rows, width // 128, 128)
    scales = np.maximum(np.abs(blocks).max(axis=2) / np.float32(448), np.float32(2.0 ** -126))
    assert scales.dtype == np.float32
    quotients = blocks / scales[..., None]
    assert quotients.dtype == np.float32
    return fp8.e4m3_codes(quotients).reshape(rows, width), np.ascontiguousarray(scales.T)


def check(device, x):
    codes, scales = run_quantize(device, x)
    want, want_scales = want_codes(x)
    assert np.array_equal(scales, want_scales)
    off = codes != want
    assert not off.any(), (int(off.sum()), x[off][:4], codes[off][:4], want[off][:4])


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_ties_at_any_scale(hip_device, dtype):
    """Blocks whose largest value is 7 k have the scale k / 64, exactly, and a tie's quotient is exact in fp32 too."""
    k = np.arange(1, 293)[:, None]
    x = np.concatenate([7.0 * k, TIES * k / 64, -TIES[:1] * k / 64], axis=1).astype(dtype)
    if dtype == "float32":
        assert np.array_equal(x[:, 1:127].astype(np.float64), TIES * k / 64)
        assert np.array_equal(want_codes(x)[0][:, 1:127],
                              np.broadcast_to(np.where(np.arange(126) % 2, np.arange(1, 127), np.arange(126)), (292, 126)))
    check(hip_device, x)


@pytest.mark.parametrize("size", [1e-41, 1e-37, 1e-35, 1e-30, 1e-27, 1e-26, 1e-20, 1.0, 1e20, 1e36])
def test_codes_of_random_values(hip_device, size):
    """The blocks' scales from the smallest one on, where they and the quotient's remainders are close to fp32's end, to the
    largest ones."""
    rng = np.random.default_rng(int(abs(np.log10(size))))
    x = rng.standard_normal((64, 1024)).astype(np.float32) * np.exp2(-rng.integers(0, 8, (64, 1024))).astype(np.float32)
    x = (x.astype(np.float64) * size * 8.0 ** rng.uniform(-1, 1, (64, 1))).astype(np.float32)
    assert np.isfinite(x).all()
    check(hip_device, x)


@pytest.mark.parametrize("size", [1e-36, 1.0, 1e30])
def test_values_next_to_ties(hip_device, size):
    """The ties of random scales as fp32 rounds them, and the values on either side."""
    rng = np.random.default_rng(3)
    top = (rng.uniform(1, 2, (96, 1)) * size).astype(np.float32)
    scale = np.maximum(top / np.float32(448), np.float32(2.0 ** -126)).astype(np.float64)
    tie = (TIES * scale).astype(np.float32)
    x = np.concatenate([np.concatenate([top, top, t], axis=1) for t in (tie, np.nextafter(tie, np.float32(0)),
                                                                        np.nextafter(tie, np.float32(np.inf)))], axis=1)
    check(hip_device, x)
    check(hip_device, -x)


def test_norm_codes_are_of_the_quotient(hip_device):
    """A norm whose results are exact (rows of one magnitude, a weight that gives the values): ties at scales k / 64."""
    k = np.arange(1, 65)
    x = np.ones((1, 128 * 64), np.float32)
    weight = np.concatenate([np.concatenate([[7.0 * j], TIES * j / 64, [0.0]]) for j in k]).astype(np.float32)
    codes, scales = run_norm(hip_device, x, None, weight, 2.0 ** -100, "codes")  # 1 / sqrt(1) = 1
    want, want_scales = want_codes(weight[None])
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, want)
