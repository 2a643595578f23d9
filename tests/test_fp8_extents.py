"""Launches of the norm and 8-bit rows past 2^32 threads are refused, those below it pass every check of their descriptors (CPU only)."""

from __future__ import annotations

import pytest

from tests.test_fp8 import norm, quantize
from tests.test_paged import ERR_ARG, ERR_PROVIDER


def refused(call, shapes):
    """Whether a call with these shapes is; the others fail at the device, which no machine has."""
    for i, (name, shape) in enumerate(shapes.items()):
        call.shape(name, shape, (i + 1) << 40)
    call.call.stream.device_ordinal = 77
    for arg in call.args:
        if arg.kind == 1:
            arg.buffer.device_ordinal = 77
    status, message = call.run()
    assert status == (ERR_ARG if "too" in message else ERR_PROVIDER), message
    return status == ERR_ARG


# rows by the threads that one takes: 16 up to 128 columns, 64 up to 512, 256 up to 8192, 1024 beyond
@pytest.mark.parametrize("width,most", [(1, (1 << 28) - 16), (128, (1 << 28) - 16), (129, (1 << 26) - 4), (8192, (1 << 24) - 1),
                                        (8193, (1 << 22) - 1)])
@pytest.mark.parametrize("codes", [False, True])
def test_rows_of_a_norm(codes, width, most):
    for rows, over in ((most, False), (most + 1, True)):
        shapes = {"x": (rows, width), "weight": (width,)}
        shapes |= {"codes": (rows, width), "scales": (-(-width // 128), rows)} if codes else {"out": (rows, width)}
        assert refused(norm(codes), shapes) == over, (rows, width)


@pytest.mark.parametrize("width,most", [(1, (1 << 28) - 16), (256, (1 << 28) - 16), (257, (1 << 27) - 16)])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_in_8_bits(gated, width, most):
    """A workgroup of 256 threads has two blocks of 16 rows."""
    for rows, over in ((most, False), (1 << 28, True)):
        shapes = {"x": (rows, width * (2 if gated else 1)), "codes": (rows, width), "scales": (-(-width // 128), rows)}
        assert refused(quantize(gated), shapes) == over, (rows, width)
