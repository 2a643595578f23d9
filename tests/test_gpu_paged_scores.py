"""Paged attention of large scores, and of rows that one key dominates."""

from __future__ import annotations

import numpy as np
import pytest

from tests.paged_cases import paging
from tests.test_gpu_paged import run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", range(16, 31, 2))
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_large_scores(hip_device, sign, power, dim):
    """Scores of 2 ** power for every dimension and so on, all of them exact: the two largest are equal and those after
    them weigh nothing, so that a row is half the sum of two values, which fp16 holds."""
    rng = np.random.default_rng(power)
    counts, lengths, prefix = [1, 3, 40], [90, 33, 70], 75
    table, shared, pages = paging(rng, lengths, 16, prefix)
    q = np.zeros((sum(counts), 4, dim), np.float16)
    q[...] = sign * 2.0 ** (power // 2) * (1.0 + np.arange(4) / 4)[:, None]
    caches = np.zeros((2, pages, 2, 16, dim), np.float16)
    caches[1] = rng.integers(-8, 9, caches[1].shape)
    levels = rng.choice([0.5, 0.625, 0.75], (pages, 2, 16))
    caches[0] = 2.0 ** (power - power // 2) * (levels if sign > 0 else 1.0 + levels / 2)[..., None]
    for at in (7, 66):  # two keys of the prefix
        caches[0, shared[at // 16], :, at % 16] = 2.0 ** (power - power // 2)
    first, second = (caches[1, shared[at // 16], :, at % 16].astype(np.float64) for at in (7, 66))
    want = np.repeat((first + second) / 2, 2, axis=0)  # two query heads of each key head
    got = run_attention(hip_device, q, caches[0], caches[1], np.cumsum([0, *counts]).astype(np.int32), lengths, table, shared, prefix)
    assert np.array_equal(got, np.broadcast_to(want, got.shape)), (got[0, :, :4], want[:, :4])
