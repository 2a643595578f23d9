"""Paged attention at 128 dimensions (and 64) where rows are looked up one by one, pages are missing or values are not finite."""

from __future__ import annotations

import numpy as np
import pytest

from tests import paged_cases as plain
from tests.test_gpu_paged import check_attention, make, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [1, 2, 4, 8])
def test_pages_below_a_load(hip_device, page, dim):
    """Decode alone (narrow tiles whose rows are looked up), then beside prompts and behind a prefix."""
    rng = np.random.default_rng(100 * page + dim)
    check_attention(hip_device, make(rng, [1, 1, 1, 2], [1, 33, 150, 64], 0, 8, 2, dim, page))
    check_attention(hip_device, make(rng, [1, 3, 70, 1], [90, 31, 100, 7], 67, 8, 2, dim, page))


@pytest.mark.parametrize("page", [1, 8, 16, 64])
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1])
def test_missing_pages(hip_device, bad, page):
    """Own pages and the prefix's that are no pages: the first, one inside, the last one."""
    rng = np.random.default_rng(page)
    for at in (0, 1, -1):
        call = make(rng, [1, 50, 2], [200, 130, 70], 140, 8, 2, 128, page)
        for row, n in zip(call[5], (200, 130, 70)):
            row[at % -(-n // page)] = bad
        call[6][at] = bad
        check_attention(hip_device, call)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("counts,lengths", [([4], [70]), ([40], [100]), ([3, 70], [3, 200])], ids=str)
def test_hidden_values_that_are_not_finite(hip_device, counts, lengths, page, value):
    """A key or value of the last token but one: nothing of it before that token, all of it from there on."""
    rng = np.random.default_rng(sum(lengths))
    clean = make(rng, counts, lengths, 20, 8, 2, 128, page)
    want, bound = plain.attention(*clean)
    b, place, d = len(counts) - 1, lengths[-1] - 2, 77
    before = int(clean[3][-1]) - 2
    for which in (1, 2):
        call = [x.copy() if isinstance(x, np.ndarray) else x for x in clean]
        call[which][clean[5][b, place // page], 0, place % page, d] = value
        got = run_attention(hip_device, *call)
        assert (np.abs(got - want)[:before] <= bound[:before]).all()
        assert (np.abs(got - want)[:, 4:] <= bound[:, 4:]).all()  # the other key head's
        if which == 2:
            assert np.array_equal(got[before:, :4, d], np.full((2, 4), value), equal_nan=True)
            rest = np.delete(np.abs(got - want) - bound, d, axis=2)
            assert (rest[before:] <= 0).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_own_keys_reach_over_several_page_windows(hip_device, dim):
    """Lists of more than 64 pages a window and 128 a ring, of one token each, read by a wave and by a workgroup."""
    rng = np.random.default_rng(dim)
    check_attention(hip_device, make(rng, [1, 2], [700, 333], 0, 4, 1, dim, 1))
    check_attention(hip_device, make(rng, [60], [500], 300, 4, 1, dim, 1))
