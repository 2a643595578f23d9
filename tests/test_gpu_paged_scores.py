"""Paged attention of large scores, and of rows that one key dominates."""

from __future__ import annotations

import math

import numpy as np
import pytest

from tests.paged_cases import paging
from tests.test_gpu_paged import Buffers, run_attention

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


LOW, SINK = 1024.0, 3.0  # values of the other keys (dimension 0) and of the first one (dimension 1)


def attend(device, octaves, *, counts, lengths, prefix, heads, kv, dim, page):
    """Rows that see a first key and, each weighing 2 ** -octaves of it, `below` others; every list of keys is made
    of two pages, so that a list of any length is a short cache.  (outputs, what a row sees besides the first key)"""
    cache = np.zeros((2, 2, kv, page, dim), np.float16)  # page 0 begins with the first key, page 1 does not
    cache[0, 0, :, 0, 0] = 16.0
    cache[1, :, :, :, 0] = LOW
    cache[1, 0, :, 0, 0], cache[1, 0, :, 0, 1] = 0.0, SINK
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = np.zeros((offsets[-1], heads, dim), np.float16)
    q[..., 0] = 1.0
    table = np.ones((len(counts), max(1, -(-max(lengths) // page))), np.int32)
    shared = np.ones(max(1, -(-prefix // page)), np.int32)
    (shared if prefix else table.T)[0] = 0  # whose first entry is the page of the first key
    below = np.concatenate([prefix - 1 + n - count + np.arange(1, count + 1) if n else np.full(count, prefix - 1)
                            for count, n in zip(counts, lengths)])
    with Buffers(device) as put:
        kernel = device.load("paged_attention", scale=octaves * math.log(2.0) / 16.0)
        workspace = put.empty((device.attention_workspace(len(q), len(counts), heads, kv, dim),), "uint8")
        out = put.empty(q.shape, "float16")
        kernel.launch(put(q), put(cache[0]), put(cache[1]), put(offsets), put(np.asarray(lengths, np.int32)), put(table),
                      put(shared), put(np.array([prefix], np.int32)), workspace, out)
        return out.to_numpy().astype(np.float64), below


def check(device, octaves, **call):
    """Each weight is rounded to fp16, 2^-11 of it, or 2^-32 of the first key's where it is below fp16's normal
    values (from 2^-21 on); a lane's sum in fp32 has a rounding, 2^-24, for every two of its keys, which are half of
    the keys or a quarter, and the product's one for every 16; scores and exponents are off by 2^-23 of the octaves."""
    got, below = attend(device, octaves, **call)
    w = 2.0 ** -octaves
    off = np.maximum(2.0 ** -11 * w, 2.0 ** -32) + w * 2.0 ** -22 * (octaves + 1)
    total = 1.0 + below * w
    sums = 2.0 ** -11 + below / 4.0 * 2.0 ** -24
    for d, want, moved in ((0, LOW * below * w / total, LOW * below * off / total), (1, SINK / total, SINK * 2.0 ** -11)):
        want = want[:, None]
        bound = np.reshape(moved, (-1, 1)) + want * ((below * off / total + sums)[:, None] + 2.0 ** -11) + 2.0 ** -25
        assert (np.abs(got[..., d] - want) <= bound).all(), (octaves, d, got[:2, :2, d], want[:2], bound[:2])
    assert (got[..., 2:] == 0).all()


OCTAVES = [9.3, 16.6, 21.5, 25.2, 27.4]


@pytest.mark.parametrize("octaves", OCTAVES)
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_of_one_tile(hip_device, dim, octaves):
    """Decode (a narrow tile of 32 keys), a prompt, and drafted tokens and a prompt behind a prefix (wide tiles of 64)."""
    size = dict(heads=8, kv=2, dim=dim, page=16)
    check(hip_device, octaves, counts=[1], lengths=[32], prefix=0, **size)
    check(hip_device, octaves, counts=[40], lengths=[60], prefix=0, **size)
    check(hip_device, octaves, counts=[5, 3], lengths=[0, 0], prefix=64, **size)
    check(hip_device, octaves, counts=[100], lengths=[100], prefix=64, **size)


@pytest.mark.parametrize("octaves", OCTAVES)
def test_keys_of_one_long_segment(hip_device, octaves):
    """As many items as ranges, so that one range holds all keys of an item: 2048 of one row and 65536 keys for the waves,
    512 of 128 rows and 32768 keys for the workgroups."""
    check(hip_device, octaves, counts=[1] * 1024, lengths=[65536] * 1024, prefix=0, heads=2, kv=2, dim=64, page=1024)
    check(hip_device, octaves, counts=[4096], lengths=[0], prefix=32768, heads=16, kv=2, dim=64, page=1024)
