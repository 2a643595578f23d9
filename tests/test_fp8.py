"""Norm and 8-bit operators without a GPU: manifests, codes and weights, and the entry points' refusals (made before any
device state is touched)."""

from __future__ import annotations

import math

import numpy as np
import pytest

from tensor_amd import _native
from tensor_amd.kernels import builtin, fp8
from tensor_amd.runtime.signature import Signature
from tests import fp8_cases as plain
from tests.test_paged import ERR_ABI, ERR_ARG, ERR_PROVIDER, Call


def test_manifests_compile_and_options_are_checked():
    for name, options in (("rms_norm", {}), ("rms_norm", {"residual": "float32", "out_dtype": "float32", "eps": 1e-5}),
                          ("rms_norm_fp8", {"dtype": "float32", "residual": "float16"}), ("rms_norm_fp8", {}),
                          ("quantize_fp8", {}), ("quantize_fp8", {"gated": True}), ("fp8_linear", {"out_dtype": "float32"})):
        manifest = builtin.manifest(name, **options)
        Signature(manifest)
        assert manifest["entrypoint"] in _native.KERNELS
    for name, options in (("rms_norm", {"dtype": "bfloat16"}), ("rms_norm", {"residual": True}), ("rms_norm", {"eps": 0.0}),
                          ("rms_norm", {"eps": -1e-6}), ("rms_norm", {"eps": math.nan}), ("rms_norm", {"eps": 1e-60}),
                          ("rms_norm", {"eps": math.inf}), ("rms_norm", {"eps": True}), ("rms_norm", {"out_dtype": "uint8"}),
                          ("quantize_fp8", {"gated": 1}), ("quantize_fp8", {"dtype": "uint8"}),
                          ("fp8_linear", {"out_dtype": "bfloat16"}), ("fp8", {})):
        with pytest.raises(ValueError):
            builtin.manifest(name, **options)
    with pytest.raises(TypeError):
        builtin.manifest("rms_norm_fp8", out_dtype="float16")


def test_shapes_follow_the_inputs():
    class Described:
        def __init__(self, *shape, dtype="float16"):
            self.shape, self.dtype = shape, dtype

    signature = Signature(builtin.manifest("quantize_fp8", gated=True))
    symbols, _ = signature.bind({"x": Described(5, 2 * 130)})
    assert signature.by_name["codes"].shape(symbols) == (5, 130) and signature.by_name["scales"].shape(symbols) == (2, 5)
    with pytest.raises(ValueError):
        signature.bind({"x": Described(5, 2 * 130 + 1)})
    signature = Signature(builtin.manifest("fp8_linear"))
    inputs = {"x": Described(3, 144, dtype="uint8"), "x_scales": Described(2, 3, dtype="float32"),
              "w": Described(129, 144, dtype="uint8"), "w_scales": Described(2, 2, dtype="float32")}
    symbols, _ = signature.bind(inputs)
    assert signature.by_name["out"].shape(symbols) == (3, 129)
    for name, other in (("x", Described(3, 152, dtype="uint8")), ("x_scales", Described(3, 2, dtype="float32")),
                        ("w_scales", Described(1, 2, dtype="float32"))):
        with pytest.raises(ValueError):
            signature.bind({**inputs, name: other})
    signature = Signature(builtin.manifest("rms_norm"))
    with pytest.raises(ValueError):
        signature.bind({"x": Described(1, 32769), "weight": Described(32769, dtype="float32")})


def test_codes():
    values = plain.value(np.arange(256))
    assert np.array_equal(fp8.e4m3_values().astype(np.float64), values, equal_nan=True)
    real = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    assert np.array_equal(fp8.e4m3_codes(values[real]), real)
    ordered = real[:127]  # ascending
    middle = (values[ordered][1:] + values[ordered][:-1]) / 2
    even = np.where(ordered[1:] % 2 == 0, ordered[1:], ordered[:-1])
    assert np.array_equal(fp8.e4m3_codes(middle), even)  # ties
    assert np.array_equal(fp8.e4m3_codes(np.nextafter(middle, 1e9)), ordered[1:])
    assert np.array_equal(fp8.e4m3_codes(-np.nextafter(middle, 0)), ordered[:-1] + 128)
    assert fp8.e4m3_codes([1e9, -1e9, math.inf, -math.inf, math.nan, 2.0 ** -11]).tolist() == [126, 254, 127, 255, 127, 0]


def test_weights_in_8_bits():
    rng = np.random.default_rng(3)
    weight = rng.standard_normal((300, 272)).astype(np.float32) * np.exp(rng.standard_normal((300, 1)))
    weight[:128, :128] = 0.0
    codes, scales = fp8.quantize_weight(weight)
    assert codes.dtype == np.uint8 and scales.dtype == np.float32 and scales.shape == (3, 3) and scales[0, 0] == 2.0 ** -126
    per_value = np.repeat(np.repeat(scales, 128, 0)[:300], 128, 1)[:, :272].astype(np.float64)
    u = weight / per_value
    assert (np.abs(plain.value(codes) - u) <= np.maximum(np.abs(u) * 2.0 ** -4, 2.0 ** -10) * (1 + 2.0 ** -20)).all()
    assert np.abs(plain.value(codes)).max() == 448.0
    for wrong in (np.zeros(4), np.zeros((0, 4)), np.full((2, 2), np.nan), np.full((2, 2), np.inf)):
        with pytest.raises(ValueError):
            fp8.quantize_weight(wrong)


# ---------------------------------------------------------------- refusals

def norm(codes=False, residual=None, **options):
    manifest = builtin.manifest("rms_norm_fp8" if codes else "rms_norm", residual=residual, **options)
    shapes = {"x": (5, 200), "residual": (5, 200), "weight": (200,), "out": (5, 200), "codes": (5, 200), "scales": (2, 5),
              "residual_out": (5, 200)}
    return Call(manifest, shapes, {})


def quantize(gated=False):
    return Call(builtin.manifest("quantize_fp8", gated=gated),
                {"x": (5, 400) if gated else (5, 200), "codes": (5, 200), "scales": (2, 5)}, {})


def linear():
    return Call(builtin.manifest("fp8_linear"),
                {"x": (5, 272), "x_scales": (3, 5), "w": (200, 272), "w_scales": (2, 3), "out": (5, 200)}, {})


CALLS = {"norm": norm, "norm_add": lambda: norm(residual="float32"), "norm_fp8": lambda: norm(True),
         "norm_fp8_add": lambda: norm(True, "float16"), "quantize": quantize, "gated": lambda: quantize(True), "linear": linear}


@pytest.mark.parametrize("name", CALLS)
def test_refusals_of_every_call(name):
    make = CALLS[name]
    call = make()
    call.call.abi_version = 2
    assert call.run()[0] == ERR_ABI
    call = make()
    call.call.argument_count += 1
    assert call.run()[0] == ERR_ARG
    call = make()
    call.call.stream.device_type = 2
    assert call.run()[0] == ERR_PROVIDER
    buffers = [a["name"] for a in make().manifest["arguments"] if a.get("kind") != "scalar"]
    for buffer in buffers:
        for field, value in (("address", 0), ("address", 0x100008), ("device_type", 1), ("device_ordinal", 1), ("rank", 3),
                             ("byte_size", 3), ("dtype", 13)):
            call = make()
            setattr(call.args[call.index[buffer]].buffer, field, value)
            assert call.run()[0] == ERR_ARG, (buffer, field)
        call = make()
        shape = [call.args[call.index[buffer]].buffer.shape[i] for i in range(call.args[call.index[buffer]].buffer.rank)]
        for axis in range(len(shape)):  # one more, or none
            if name in ("quantize", "gated") and buffer == "x" and axis == 1:
                continue  # (below)
            for extent in (shape[axis] + 1, 0):
                call = make()
                call.shape(buffer, [extent if i == axis else n for i, n in enumerate(shape)])
                assert call.run()[0] == ERR_ARG, (buffer, axis)
        call = make()
        strides = call.args[call.index[buffer]].buffer.strides
        strides[0] += 16
        assert call.run()[0] == ERR_ARG, buffer
    scalars = [a["name"] for a in make().manifest["arguments"] if a.get("kind") == "scalar"]
    for scalar in scalars:
        call = make()
        call.args[call.index[scalar]].dtype = 6
        assert call.run()[0] == ERR_ARG
        call = make()
        call.args[call.index[scalar]].scalar |= 1 << 40
        assert call.run()[0] == ERR_ARG


def test_refusals_of_values():
    for bits in (0, 0x80000000, 0x7F800000, 0x7FC00000, 0xBF800000):  # 0, -0, infinity, NaN, -1
        call = norm()
        call.args[call.index["eps"]].scalar = bits
        status, message = call.run()
        assert status == ERR_ARG and "eps" in message
    call = quantize()
    call.args[call.index["gated"]].scalar = 2
    assert call.run()[0] == ERR_ARG
    call = quantize(True)
    call.shape("x", (5, 401))
    assert call.run()[0] == ERR_ARG


def test_least_eps():
    assert builtin.manifest("rms_norm", eps=2.0 ** -100)
    with pytest.raises(ValueError, match="eps"):
        builtin.manifest("rms_norm", eps=2.0 ** -101)
    call = norm()
    call.args[call.index["eps"]].scalar = int(np.float32(2.0 ** -101).view(np.uint32))
    status, message = call.run()
    assert status == ERR_ARG and "eps" in message


def test_refusals_of_sizes():
    call = norm()
    for name, shape in (("x", (1, 32769)), ("weight", (32769,)), ("out", (1, 32769))):
        call.shape(name, shape)
    assert call.run()[0] == ERR_ARG
    call = norm()
    for name, shape in (("x", (1 << 31, 4)), ("weight", (4,)), ("out", (1 << 31, 4))):
        call.shape(name, shape, 1 << 44 if name == "out" else None)
    assert call.run()[0] == ERR_ARG
    call = linear()
    for name, shape in (("x", (5, 264)), ("w", (200, 264))):  # no multiple of 16 columns
        call.shape(name, shape)
    assert call.run()[0] == ERR_ARG
    for m, n, k in (((1 << 20) + 1, 16, 16), (1, (1 << 22) + 1, 16), (1, 16, (1 << 20) + 16)):
        call = linear()
        for i, (name, shape) in enumerate((("x", (m, k)), ("x_scales", (-(-k // 128), m)), ("w", (n, k)),
                                           ("w_scales", (-(-n // 128), -(-k // 128))), ("out", (m, n)))):
            call.shape(name, shape, (i + 1) << 44)
        assert call.run()[0] == ERR_ARG, (m, n, k)


WRITTEN = [("norm", "out", "weight", 0), ("norm", "out", "x", 16), ("norm_add", "out", "residual", 0),
           ("norm_add", "residual_out", "out", 0), ("norm_add", "residual_out", "x", 0), ("norm_add", "residual_out", "residual", 16),
           ("norm_fp8", "codes", "x", 0), ("norm_fp8", "scales", "weight", 0), ("norm_fp8_add", "residual_out", "codes", 0),
           ("norm_fp8_add", "scales", "codes", 0), ("quantize", "codes", "x", 0), ("quantize", "scales", "codes", 16),
           ("gated", "codes", "x", 0), ("linear", "out", "x", 0), ("linear", "out", "w", 16), ("linear", "out", "x_scales", 0),
           ("linear", "out", "w_scales", 0)]


@pytest.mark.parametrize("case", WRITTEN, ids=str)
def test_written_buffers_stand_apart(case):
    name, written, other, offset = case
    call = CALLS[name]()
    call.args[call.index[written]].buffer.address = call.args[call.index[other]].buffer.address + offset
    status, message = call.run()
    assert status == ERR_ARG and "shares memory" in message


def test_outputs_that_may_be_inputs_pass_the_checks():
    """They get past every descriptor check: without a GPU the next one, of the device, fails."""
    for name, written, other in (("norm", "out", "x"), ("norm_add", "residual_out", "residual"), ("norm_add", "out", "x")):
        call = CALLS[name]()
        call.call.stream.device_ordinal = 77  # no device has it, with a GPU or without
        for arg in call.args:
            if arg.kind == 1:
                arg.buffer.device_ordinal = 77
        call.args[call.index[written]].buffer.address = call.args[call.index[other]].buffer.address
        status, message = call.run()
        assert status == ERR_PROVIDER, message
    call = norm(dtype="float32")  # fp16 results over fp32 values
    call.args[call.index["out"]].buffer.address = call.args[call.index["x"]].buffer.address
    assert call.run()[0] == ERR_ARG
