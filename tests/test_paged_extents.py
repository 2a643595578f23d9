"""Paged-cache calls whose launches would pass 2^32 threads: refused like any other extent, before device state is
touched (CPU only, on fake addresses)."""

from __future__ import annotations

import pytest

from tensor_amd.kernels import builtin
from tests.test_paged import ERR_ARG, ERR_PROVIDER, Call, workspace
from tests.test_paged_apart import spread


def far(call):
    """The call on a device that no machine has, its buffers apart."""
    call = spread(None, call)
    for i, arg in enumerate(call.args):
        if arg.kind == 1:
            arg.buffer.address = (i + 1) << 42
    return call.run()


def slots(requests):
    shapes = dict(lengths=(requests,), counts=(requests,), start=(1,), free=(9,), free_count=(1,), table=(requests, 1),
                  offsets=(requests + 1,), lengths_out=(requests,), positions=(4,), slots=(4,), table_out=(requests, 1), free_left=(1,))
    return Call(builtin.manifest("paged_slots", page_size=16), shapes, dict(T=4))


def rotary(tokens, heads, kv, dim, store=False):
    shapes = dict(q=(tokens, heads, dim), k=(tokens, kv, dim), v=(tokens, kv, dim), positions=(tokens,), slots=(tokens,),
                  angles=(10, 2), q_out=(tokens, heads, dim), k_out=(tokens, kv, dim), k_cache=(5, kv, 16, dim), v_cache=(5, kv, 16, dim))
    return Call(builtin.manifest("rotary_store" if store else "rotary"), shapes, {})


def attention(tokens, heads, kv, dim):
    shapes = dict(q=(tokens, heads, dim), k_cache=(5, kv, 16, dim), v_cache=(5, kv, 16, dim), offsets=(3,), lengths=(2,),
                  table=(2, 4), prefix_pages=(1,), prefix_length=(1,), workspace=(1 << 40,), out=(tokens, heads, dim))
    return Call(builtin.manifest("paged_attention"), shapes, {})


@pytest.mark.parametrize("fits,passes,name", [
    (slots((1 << 24) - 1), slots(1 << 24), "lengths"),
    # workgroups of 64 threads, and of 256
    (rotary((1 << 26) - 1, 1, 1, 2), rotary(1 << 26, 1, 1, 2), "q"),
    (rotary((1 << 26) - 1, 1, 1, 2, True), rotary(1 << 26, 1, 1, 2, True), "q"),
    (rotary((1 << 24) - 1, 255, 1, 2), rotary(1 << 24, 255, 1, 2), "q"),
    (attention(4095, 1 << 15, 1 << 15, 128), attention(4096, 1 << 15, 1 << 15, 128), "q"),
    (attention(8191, 1 << 15, 1 << 15, 64), attention(8192, 1 << 15, 1 << 15, 64), "q")], ids=range(6))
def test_threads_of_a_launch(fits, passes, name):
    status, message = far(fits)
    assert status == ERR_PROVIDER, message
    status, message = far(passes)
    assert status == ERR_ARG and message.startswith(name), message


def test_workspace_query_takes_the_same_extents():
    assert workspace((1 << 20) - 1, 1, 128, 8, 128)[0] == 0
    assert workspace(1 << 20, 1, 128, 8, 128)[0] == ERR_ARG
