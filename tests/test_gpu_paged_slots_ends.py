"""Slot maps whose sums pass int32: held at its end, where a wrapped one would be a length of 0 or padding."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_paged import run_slots

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("page", [1, 16, 1024])
def test_lengths_and_positions_stop_at_the_end_of_int32(hip_device, page):
    table = np.full((4, 3), 7)
    offsets, lengths, positions, slots, out, left = run_slots(
        hip_device, [TOP, TOP - 2, TOP - 9, 0], [1, 3, 2, 2], 100, [5], 1, table, 8, page)
    assert offsets.tolist() == [0, 1, 4, 6, 8]
    assert lengths.tolist() == [TOP, TOP, TOP - 7, 2]
    assert positions.tolist() == [TOP] * 6 + [100, 101]
    assert (slots[:6] == -1).all() and (out[:3] == 7).all() and left.tolist() == [0 if page > 1 else -1]


def test_positions_of_a_negative_start(hip_device):
    *_, positions, slots, _, _ = run_slots(hip_device, [3], [4], -5, [1], 0, np.array([[2, 4]]), 4, 4)
    assert positions.tolist() == [-2, -1, 0, 1] and slots.tolist() == [11, -1, -1, -1]
