"""Paged-cache operators on buffers that are both read and written."""

from __future__ import annotations

import numpy as np
import pytest

from tests import paged_cases as plain
from tests.test_gpu_paged import Buffers

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
