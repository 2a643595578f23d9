"""The transposed rotary map on a table whose cosines and sines are scaled: the gradient, not the inverse."""

from __future__ import annotations

import numpy as np
import pytest

from tensor_amd.kernels.paged import rotary_angles
from tests import paged_cases as plain
from tests.test_gpu_paged import Buffers, bound_rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rotated", [32, 20])
def test_gradient_on_a_scaled_table(hip_device, rotated, layout):
    """Of sum(g * rotary(x)), against central differences of the 64-bit form (the map is linear: exact but for their
    rounding); and there and back is the square of the scale."""
    rng = np.random.default_rng(rotated)
    tokens, heads, dim = 5, 3, 32
    angles = rotary_angles(300, rotated, scaling="yarn", factor=4.0, original=64)
    positions = np.array([0, 1, 17, 150, 299], np.int32)
    x, g = (rng.standard_normal((tokens, heads, dim)).astype(np.float32) for _ in range(2))
    with Buffers(hip_device) as put:
        forward, back = (hip_device.load("rotary", layout=layout, dtype="float32", inverse=inverse) for inverse in (False, True))
        at, table = put(positions), put(angles)
        turned, gradient, again = ([put.empty(x.shape, "float32") for _ in range(2)] for _ in range(3))
        forward.launch(put(x), put(x), at, table, *turned)
        back.launch(put(g), put(g), at, table, *gradient)
        back.launch(*turned, at, table, *again)
        turned, gradient, again = (b[1].to_numpy().astype(np.float64) for b in (turned, gradient, again))
    assert (np.abs(turned - plain.rotary(x, positions, angles, layout)) <= bound_rotary(x, angles, "float32")).all()
    bound = bound_rotary(g, angles, "float32")[..., 0] + 1e-12
    for d in range(dim):
        step = np.zeros_like(x, np.float64)
        step[..., d] = 0.5
        change = (g * (plain.rotary(x + step, positions, angles, layout) - plain.rotary(x - step, positions, angles, layout))).sum(-1)
        assert (np.abs(gradient[..., d] - change) <= bound).all()
    pairs = rotated // 2
    square = angles[positions, :pairs].astype(np.float64) ** 2 + angles[positions, pairs:].astype(np.float64) ** 2
    scale = np.ones((tokens, dim))
    scale[:, :rotated] = np.concatenate([square, square], 1) if layout == "half" else np.repeat(square, 2, axis=1)
    # the second map's rounding, of values as large as the first one's, and the first one's carried through it
    carried = bound_rotary(turned, angles, "float32") + 2.0 * np.abs(angles).max() * bound_rotary(x, angles, "float32")
    assert (np.abs(again - scale[:, None] * x) <= carried).all()
    assert np.abs(again[..., :rotated] / x[..., :rotated]).min() > 1.2  # f^2 = 1.297
