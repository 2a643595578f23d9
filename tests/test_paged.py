"""Paged-cache operators without a GPU: manifests, the angle table, and the entry points' refusals (made
before any device state is touched)."""

from __future__ import annotations

import ctypes as c
import math

import numpy as np
import pytest

from tensor_amd import _native
from tensor_amd.kernels import builtin, paged
from tensor_amd.runtime import abi
from tensor_amd.runtime.signature import Signature

DTYPES = {"uint8": (3, 1), "int32": (6, 4), "uint32": (7, 4), "float16": (10, 2), "float32": (11, 4)}
ERR_ABI, ERR_ARG, ERR_PROVIDER = 1, 2, 3


def test_manifests_compile_and_options_are_checked():
    for name, options in (("paged_slots", {"page_size": 16}), ("rotary", {}), ("rotary_store", {"layout": "interleaved"}),
                          ("paged_attention", {"scale": 0.25})):
        manifest = builtin.manifest(name, **options)
        Signature(manifest)
        assert manifest["entrypoint"] in _native.KERNELS
    assert builtin.manifest("gguf_linear", encoding="q4_k")["entrypoint"] == "tensor_gguf_linear_v1"
    for name, options in (("paged_slots", {"page_size": 24}), ("paged_slots", {"page_size": 2048}), ("rotary", {"layout": "x"}),
                          ("rotary", {"dtype": "bfloat16"}), ("rotary", {"inverse": 1}), ("paged_attention", {"scale": 0.0}),
                          ("paged_attention", {"scale": -1.0}), ("paged_attention", {"scale": math.inf}),
                          ("paged_attention", {"scale": 1e-60}), ("paged_attention", {"scale": True}), ("paged", {})):
        with pytest.raises(ValueError):
            builtin.manifest(name, **options)


# ------------------------------------------------------------------ angles

def test_angles():
    table = paged.rotary_angles(70000, 8, base=10000.0)
    assert table.shape == (70000, 8) and table.dtype == np.float32
    for position in (0, 1, 69999):
        for pair in range(4):
            angle = position * 10000.0 ** (-pair / 4)
            assert abs(table[position, pair] - math.cos(angle)) < 1e-7
            assert abs(table[position, 4 + pair] - math.sin(angle)) < 1e-7


def test_scaled_angles():
    plain = paged.rotary_angles(64, 16, base=1e4)
    linear = paged.rotary_angles(256, 16, base=1e4, scaling="linear", factor=4.0)
    assert np.abs(linear[::4] - plain).max() < 1e-6  # position 4 p turns as p did
    ntk = paged.rotary_angles(256, 16, base=1e4, scaling="ntk", factor=4.0)
    assert np.abs(ntk[:64, 0] - plain[:, 0]).max() < 1e-6                   # the fastest pair is kept
    assert np.abs(ntk[::4, 7] - plain[:, 7]).max() < 1e-6                   # the slowest is slowed by the factor
    yarn = paged.rotary_angles(256, 16, base=1e4, scaling="yarn", factor=4.0, original=512) / (0.1 * math.log(4.0) + 1.0)
    assert np.abs(yarn[:64, 0] - plain[:, 0]).max() < 1e-6
    assert np.abs(yarn[::4, 7] - plain[:, 7]).max() < 1e-6
    assert np.abs(paged.rotary_angles(64, 16, scaling="yarn", factor=1.0, original=64) - plain).max() < 1e-6


@pytest.mark.parametrize("arguments", [
    dict(reach=0, rotated=8), dict(reach=8, rotated=7), dict(reach=8, rotated=0), dict(reach=8.0, rotated=8),
    dict(reach=8, rotated=8, base=1.0), dict(reach=8, rotated=8, base=math.nan), dict(reach=8, rotated=8, factor=2.0),
    dict(reach=8, rotated=8, scaling="linear", factor=0.5), dict(reach=8, rotated=8, scaling="cubic"),
    dict(reach=8, rotated=2, scaling="ntk", factor=2.0), dict(reach=8, rotated=8, scaling="yarn", factor=2.0),
    dict(reach=8, rotated=8, scaling="yarn", factor=2.0, original=64, fast=1.0, slow=2.0)], ids=str)
def test_angles_refuse(arguments):
    with pytest.raises(ValueError):
        paged.rotary_angles(arguments.pop("reach"), arguments.pop("rotated"), **arguments)


# ---------------------------------------------------------------- refusals

class Call:
    """A well-formed call of a manifest on fake (never dereferenced) addresses."""

    def __init__(self, manifest, shapes, scalars):
        self.manifest, self.keep = manifest, []
        arguments = manifest["arguments"]
        self.args = (abi.Argument * len(arguments))()
        self.index = {a["name"]: i for i, a in enumerate(arguments)}
        values = {**manifest["constants"], **scalars}
        for i, a in enumerate(arguments):
            code, item = DTYPES[a["dtype"]]
            self.args[i].dtype = code
            if a.get("kind") == "scalar":
                self.args[i].kind = 2
                self.args[i].scalar = abi._scalar_bits(values[a["name"]], a["dtype"])
            else:
                self.args[i].kind = 1
                self.shape(a["name"], shapes[a["name"]], 0x100000 * (i + 1))
        self.call = abi.CallDescriptor(1, 72, self.args, len(arguments), 0, (c.c_uint32 * 3)(1, 1, 1),
                                       (c.c_uint32 * 3)(256, 1, 1), 0, abi.StreamDescriptor(10, 0, 0))

    def shape(self, name, shape, address=None):
        arg = self.args[self.index[name]]
        item = next(size for code, size in DTYPES.values() if code == arg.dtype)
        strides, step = [], item
        for extent in reversed(shape):
            strides.insert(0, step)
            step *= extent
        arrays = (c.c_int64 * len(shape))(*shape), (c.c_int64 * len(shape))(*strides)
        self.keep.append(arrays)
        arg.buffer = abi.BufferDescriptor(address or arg.buffer.address, step, *arrays, len(shape), arg.dtype, 10, 0)

    def run(self):
        error = abi.ErrorDescriptor()
        status = _native.kernel(self.manifest["entrypoint"])(c.byref(self.call), c.byref(error))
        return status, error.message.decode()


def slots_call():
    return Call(builtin.manifest("paged_slots", page_size=16),
                dict(lengths=(3,), counts=(3,), start=(1,), free=(9,), free_count=(1,), table=(3, 5), offsets=(4,),
                     lengths_out=(3,), positions=(4,), slots=(4,), table_out=(3, 5), free_left=(1,)), dict(T=4))


def rotary_call(store=False):
    shapes = dict(q=(3, 8, 64), k=(3, 2, 64), v=(3, 2, 64), positions=(3,), slots=(3,), angles=(10, 32), q_out=(3, 8, 64),
                  k_out=(3, 2, 64), k_cache=(5, 2, 16, 64), v_cache=(5, 2, 16, 64))
    return Call(builtin.manifest("rotary_store" if store else "rotary"), shapes, {})


def attention_call(**more):
    shapes = dict(q=(3, 8, 64), k_cache=(5, 2, 16, 64), v_cache=(5, 2, 16, 64), offsets=(3,), lengths=(2,), table=(2, 4),
                  prefix_pages=(1,), prefix_length=(1,), workspace=(1 << 26,), out=(3, 8, 64))
    return Call(builtin.manifest("paged_attention"), {**shapes, **more}, {})


CALLS = {"slots": slots_call, "rotary": rotary_call, "store": lambda: rotary_call(True), "attention": attention_call}


def refused(call, status=ERR_ARG, text=""):
    got, message = call.run()
    assert got == status and text in message, (got, message)


@pytest.mark.parametrize("kind", CALLS)
def test_descriptor_faults_are_refused(kind):
    make = CALLS[kind]
    names = [a["name"] for a in make().manifest["arguments"] if a.get("kind") != "scalar"]
    call = make()
    call.call.abi_version = 2
    refused(call, ERR_ABI)
    call = make()
    call.call.argument_count -= 1
    refused(call)
    call = make()
    call.call.stream.device_type = 2
    refused(call, ERR_PROVIDER)
    for name in names:
        for change in ("address", "align", "rank", "stride", "size", "device", "ordinal", "dtype", "kind", "extent"):
            call = make()
            arg = call.args[call.index[name]]
            if change == "address":
                arg.buffer.address = 0
            elif change == "align":
                arg.buffer.address += 2
            elif change == "rank":
                arg.buffer.rank += 1
            elif change == "stride":
                arg.buffer.strides[arg.buffer.rank - 1] *= 2
            elif change == "size":
                arg.buffer.byte_size -= 1
            elif change == "device":
                arg.buffer.device_type = 2
            elif change == "ordinal":
                arg.buffer.device_ordinal = 1
            elif change == "dtype":
                arg.buffer.dtype = 9
            elif change == "kind":
                arg.kind = 2
            else:
                call.shape(name, [0] + list(arg.buffer.shape[i] for i in range(1, arg.buffer.rank)))
            status, message = call.run()
            assert status == ERR_ARG and name in message, (name, change, status, message)


@pytest.mark.parametrize("kind", CALLS)
def test_extents_that_disagree_are_refused(kind):
    make = CALLS[kind]
    free = {"slots": ("free",), "rotary": (), "store": (), "attention": ("workspace", "prefix_pages")}[kind]
    fixed = {"angles", "k_cache", "v_cache", "table", "q"}  # extents of their own, tested below
    for a in make().manifest["arguments"]:
        if a.get("kind") == "scalar" or a["name"] in free or a["name"] in fixed:
            continue
        call = make()
        arg = call.args[call.index[a["name"]]]
        shape = [arg.buffer.shape[i] for i in range(arg.buffer.rank)]
        call.shape(a["name"], [shape[0] + 1, *shape[1:]])
        assert call.run()[0] == ERR_ARG, a["name"]


def test_slots_refusals():
    for name, value in (("page_size", 0), ("page_size", 12), ("page_size", 2048), ("T", 0), ("T", 1 << 31), ("T", 1 << 40)):
        call = slots_call()
        call.args[call.index[name]].scalar = value
        refused(call, text=name)


def test_rotary_refusals():
    for columns in (31, 66):
        call = rotary_call()
        call.shape("angles", (10, columns))
        refused(call, text="angles")
    for name in ("layout", "inverse"):
        call = rotary_call()
        call.args[call.index[name]].scalar = 2
        refused(call, text=name)
    call = rotary_call()
    call.args[0].dtype = call.args[0].buffer.dtype = 3
    refused(call, text="q")
    call = rotary_call()  # keys of another type than the queries
    call.args[1].dtype = call.args[1].buffer.dtype = 11
    refused(call, text="k")
    for cache in ((5, 2, 12, 64), (5, 3, 16, 64), (5, 2, 16, 32), (5, 2, 2048, 64)):
        call = rotary_call(True)
        call.shape("k_cache", cache)
        call.shape("v_cache", cache)
        refused(call, text="k_cache")
    call = rotary_call()
    for name, heads in (("q", 9000), ("q_out", 9000)):
        call.shape(name, (3, heads, 4096))
    for name in ("k", "k_out"):
        call.shape(name, (3, 2, 4096))
    refused(call, text="heads")


def test_attention_refusals():
    refused(attention_call(q=(3, 8, 96), out=(3, 8, 96), k_cache=(5, 2, 16, 96), v_cache=(5, 2, 16, 96)), text="64 or 128")
    refused(attention_call(q=(3, 7, 64), out=(3, 7, 64)), text="heads")
    refused(attention_call(q=(3, 258, 64), out=(3, 258, 64)), text="heads")
    refused(attention_call(offsets=(1026,), lengths=(1025,), table=(1025, 4)), text="requests")
    refused(attention_call(offsets=(1,)), text="requests")
    refused(attention_call(q=((1 << 20) + 1, 8, 64), out=((1 << 20) + 1, 8, 64)), text="tokens")
    refused(attention_call(k_cache=(5, 2, 24, 64), v_cache=(5, 2, 24, 64)), text="k_cache")
    refused(attention_call(k_cache=(5, 2, 2048, 64), v_cache=(5, 2, 2048, 64)), text="k_cache")
    refused(attention_call(table=(2, (1 << 20) + 1)), text="2^24")
    refused(attention_call(prefix_pages=((1 << 20) + 1,)), text="2^24")
    refused(attention_call(q=(1 << 19, 8, 64), out=(1 << 19, 8, 64), table=(2, 1 << 20)), text="too many")
    refused(attention_call(workspace=(4096,)), text="workspace")
    for bits in (0x7F800000, 0x7FC00000, 0xBF800000, 1 << 32):
        call = attention_call()
        call.args[call.index["scale"]].scalar = bits
        refused(call, text="scale")
    call = attention_call()
    call.args[call.index["workspace"]].buffer.address += 16
    refused(call, text="workspace")


def workspace(*sizes):
    result, error = c.c_uint64(), abi.ErrorDescriptor()
    status = _native.library().tensor_paged_attention_workspace_v1(*sizes, c.byref(result), c.byref(error))
    return status, result.value, error.message.decode()


def test_attention_workspace():
    status, small, _ = workspace(1, 1, 32, 8, 128)
    assert status == 0 and small > 0
    assert workspace(4096, 64, 32, 8, 128)[1] > small
    for sizes in ((0, 1, 32, 8, 128), (1, 0, 32, 8, 128), (1, 1025, 32, 8, 128), (1, 1, 30, 8, 128), (1, 1, 32, 0, 128),
                  (1, 1, 32, 8, 80), (1 << 21, 1, 32, 8, 128), (1, 1, 129, 1, 64), (1, 1, -8, -1, 64)):
        assert workspace(*sizes)[0] == ERR_ARG, sizes
