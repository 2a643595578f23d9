"""The rotary angle table where its frequencies are scaled one by one (CPU only)."""

from __future__ import annotations

import math

import numpy as np
import pytest

from tensor_amd.kernels.paged import rotary_angles


@pytest.mark.parametrize("rotated,base,factor,original,fast,slow", [
    (128, 1e4, 4.0, 4096, 32.0, 1.0), (64, 1e6, 8.0, 32768, 32.0, 1.0), (96, 5e5, 2.5, 8192, 16.0, 2.0), (16, 1e4, 4.0, 64, 32.0, 1.0)])
def test_yarn_between_its_ends(rotated, base, factor, original, fast, slow):
    """Every pair against the ramp written out: kept up to the pair that makes `fast` turns in the original length (rounded
    down), slowed by the factor from the one that makes `slow` on (rounded up), between them in equal steps."""
    def pair_at(turns):  # base ** (-2 p / rotated) * original = 2 pi turns
        return rotated / 2 * math.log(original / (2 * math.pi * turns), base)

    low, high = max(0, math.floor(pair_at(fast))), min(rotated - 1, math.ceil(pair_at(slow)))
    table = rotary_angles(50, rotated, base=base, scaling="yarn", factor=factor, original=original, fast=fast, slow=slow)
    between = 0
    for pair in range(rotated // 2):
        slowed = 0.0 if pair <= low else 1.0 if pair >= high else (pair - low) / (high - low)
        between += 0.0 < slowed < 1.0
        turn = base ** (-2 * pair / rotated) * ((1 - slowed) + slowed / factor)
        for position in (0, 1, 7, 49):
            for at, want in ((pair, math.cos(position * turn)), (rotated // 2 + pair, math.sin(position * turn))):
                # fp32's rounding of values up to f, and 64 bits' of angles up to 50
                assert abs(table[position, at] - (0.1 * math.log(factor) + 1) * want) <= 2.0 ** -24 * 1.25 + 1e-12
    assert between > 0
    assert table.dtype == np.float32
