"""Paged-cache operators on buffers that are both read and written."""

from __future__ import annotations

import numpy as np
import pytest

from tensor_amd.kernels.paged import rotary_angles
from tests import paged_cases as plain
from tests.test_gpu_paged import Buffers, make, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,columns,tokens", [(3, 5, 9), (300, 9, 700), (2, 9001, 20000)])
def test_slots_update_their_table_in_place(hip_device, requests, columns, tokens):
    rng = np.random.default_rng(requests)
    page = 4
    lengths = rng.integers(0, page * columns // 2, requests)
    counts = rng.multinomial(tokens, np.full(requests, 1.0 / requests))
    table, free = rng.integers(0, 1 << 20, (requests, columns)), rng.permutation(tokens)
    want = plain.slots(lengths, counts, 7, free, tokens, table, tokens, page)
    with Buffers(hip_device) as put:
        kernel = hip_device.load("paged_slots", page_size=page)
        ins = [put(np.asarray(v, np.int32)) for v in (lengths, counts, [7], free, [tokens], table)]
        outs = [put.empty((n,), "int32") for n in (requests + 1, requests, tokens, tokens)]
        left = put.empty((1,), "int32")
        kernel.launch(*ins, tokens, *outs, ins[5], left)
        for got, expected in zip((*outs, ins[5], left), want):
            assert np.array_equal(got.to_numpy(), expected)


def test_slots_refuse_their_other_inputs_as_outputs(hip_device):
    with Buffers(hip_device) as put:
        kernel = hip_device.load("paged_slots", page_size=4)
        ins = [put(np.asarray(v, np.int32)) for v in ([3, 1], [1, 1], [0], [5, 6], [2], [[0, -1], [1, -1]])]
        outs = [put.empty(shape, "int32") for shape in ((3,), (2,), (2,), (2,), (2, 2), (1,))]
        for at, which in ((1, 0), (5, 4)):  # lengths, the count of free pages
            mixed = list(outs)
            mixed[at] = ins[which]
            with pytest.raises(Exception, match="shares memory"):
                kernel.launch(*ins, 2, *mixed)
        assert [b.to_numpy().tolist() for b in ins] == [[3, 1], [1, 1], [0], [5, 6], [2], [[0, -1], [1, -1]]]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotated", [(128, 128), (64, 32), (96, 46)])
def test_store_turns_queries_in_place(hip_device, dim, rotated, layout):
    rng = np.random.default_rng(dim)
    tokens, heads, kv = 37, 6, 2
    q, k, v = (rng.standard_normal((tokens, n, dim)).astype(np.float16) for n in (heads, kv, kv))
    at, slots = rng.integers(0, 90, tokens).astype(np.int32), rng.permutation(48)[:tokens].astype(np.int32)
    with Buffers(hip_device) as put:
        kernel = hip_device.load("rotary_store", layout=layout)
        shared = [put(x) for x in (q, k, v, at, slots, rotary_angles(90, rotated))]
        caches = [put(np.zeros((3, kv, 16, dim), np.float16)) for _ in range(2)]
        apart = put.empty(q.shape, "float16")
        kernel.launch(*shared, apart, *caches)
        kernel.launch(*shared, shared[0], *caches)
        assert np.array_equal(apart.to_numpy(), shared[0].to_numpy())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(8, 2), (7, 1), (32, 1)])
def test_attention_writes_over_its_queries(hip_device, heads, kv, dim):
    """Requests of one segment, which write their rows themselves, and of many, which are joined."""
    rng = np.random.default_rng(heads + dim)
    for counts, lengths, prefix in (([1, 3, 40, 1], [9, 300, 150, 30], 0), ([1, 200, 2], [1, 200, 900], 70), ([130], [400], 0)):
        call = make(rng, counts, lengths, prefix, heads, kv, dim, 16, padding=2)
        want = run_attention(hip_device, *call)
        with Buffers(hip_device) as put:
            ins = [put(x) for x in call[:7]] + [put(np.array([prefix], np.int32))]
            need = hip_device.attention_workspace(len(call[0]), len(counts), heads, kv, dim)
            hip_device.load("paged_attention").launch(*ins, put.empty((need,), "uint8"), ins[0])
            assert np.array_equal(ins[0].to_numpy().astype(np.float64), want)
