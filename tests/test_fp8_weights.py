"""What a weight's codes and scales cannot hold is refused (CPU only)."""

from __future__ import annotations

import numpy as np
import pytest

from tensor_amd.kernels import fp8
from tests import fp8_cases as plain

FLOAT_MAX = float(np.finfo(np.float32).max)


@pytest.mark.parametrize("size", [1e300, 1e42, 448.001 * FLOAT_MAX])
@pytest.mark.parametrize("sign", [1, -1])
def test_magnitudes_past_the_largest_scale_are_refused(size, sign):
    """Their scale would be infinite and each code 0."""
    weight = np.ones((3, 200))
    weight[1, 150] = sign * size
    with pytest.raises(ValueError, match="scale"):
        fp8.quantize_weight(weight)


def test_magnitudes_up_to_the_largest_scale():
    weight = np.array([[447.999 * FLOAT_MAX, -200 * FLOAT_MAX]])
    codes, scales = fp8.quantize_weight(weight)
    assert np.isfinite(scales).all()
    assert np.allclose(plain.value(codes) * scales.astype(np.float64), weight, rtol=2.0 ** -4)


def test_complex_weights_are_refused():
    """Their imaginary parts would be lost."""
    with pytest.raises(ValueError, match="real numbers"):
        fp8.quantize_weight(np.full((2, 2), 1 + 2j))


@pytest.mark.parametrize("dtype", ["float16", "float32", "float64", "int8", "int64", "uint8"])
def test_types_of_real_numbers(dtype):
    weight = np.array([[1, 7], [100, 3]], dtype)
    codes, scales = fp8.quantize_weight(weight)
    assert scales[0, 0] == np.float32(100 / 448)
    u = weight.astype(np.float64) / float(scales[0, 0])
    assert (np.abs(plain.value(codes) - u) <= u * 2.0 ** -4).all()
