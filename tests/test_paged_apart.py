"""Paged-cache calls whose written buffers share memory with their others: refused before any device state is touched
(CPU only, on fake addresses)."""

from __future__ import annotations

import pytest

from tensor_amd.kernels import builtin
from tests.test_paged import CALLS, ERR_ARG, ERR_PROVIDER, Call

# written argument -> the input that it may be itself
WRITTEN = {"slots": {"offsets": None, "lengths_out": None, "positions": None, "slots": None, "table_out": "table",
                     "free_left": None},
           "rotary": {"q_out": "q", "k_out": "k"}, "store": {"q_out": "q", "k_cache": None, "v_cache": None},
           "attention": {"workspace": None, "out": "q"}}


def spread(kind, call=None):
    """A call whose buffers share nothing, on a device that no machine has: past the checks it ends there."""
    call = call or CALLS[kind]()
    call.call.stream.device_ordinal = 1 << 20
    for i, arg in enumerate(call.args):
        if arg.kind == 1:
            arg.buffer.address = (i + 1) << 32
            arg.buffer.device_ordinal = 1 << 20
    return call


def buffers(call):
    return [name for name, i in call.index.items() if call.args[i].kind == 1]


@pytest.mark.parametrize("kind", WRITTEN)
def test_buffers_apart_pass_the_checks(kind):
    status, message = spread(kind).run()
    assert status == ERR_PROVIDER, message
    call = spread(kind)  # next to each other
    end = 1 << 32
    for name in buffers(call):
        buffer = call.args[call.index[name]].buffer
        end = (end + 255) // 256 * 256
        buffer.address, end = end, end + buffer.byte_size
    assert call.run()[0] == ERR_PROVIDER


@pytest.mark.parametrize("kind", WRITTEN)
def test_shared_memory_is_refused(kind):
    for name in WRITTEN[kind]:
        for other in buffers(spread(kind)):
            if other == name:
                continue
            for part in ("same", "first byte", "last byte"):
                call = spread(kind)
                mine, its = (call.args[call.index[n]].buffer for n in (name, other))
                if part == "same":
                    its.address = mine.address
                elif part == "first byte":  # the other's first bytes are the written one's last
                    mine.address = its.address - (mine.byte_size - 1) // 256 * 256
                else:
                    its.address = mine.address - (its.byte_size - 1) // 256 * 256
                allowed = WRITTEN[kind][name] == other and mine.address == its.address
                status, message = call.run()
                assert status == (ERR_PROVIDER if allowed else ERR_ARG), (name, other, part, message)
                if not allowed:
                    assert "shares memory" in message and (name in message or other in message), message


def test_fp16_queries_do_not_go_into_the_fp32_ones():
    """rotary_store rounds its queries: in place, a token's would lie over another's that is still to be read."""
    shapes = dict(q=(3, 8, 64), k=(3, 2, 64), v=(3, 2, 64), positions=(3,), slots=(3,), angles=(10, 32), q_out=(3, 8, 64),
                  k_cache=(5, 2, 16, 64), v_cache=(5, 2, 16, 64))
    call = spread("store", Call(builtin.manifest("rotary_store", dtype="float32"), shapes, {}))
    assert call.run()[0] == ERR_PROVIDER
    call.args[call.index["q_out"]].buffer.address = call.args[call.index["q"]].buffer.address
    status, message = call.run()
    assert status == ERR_ARG and "shares memory" in message
