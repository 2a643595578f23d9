"""Manifests of the norm and the 8-bit operators (include/tensor_hip.h), and their weights.

They run a decoder layer around its attention when its linears are held in 8 bits, and are loaded by name as the GGUF
kernels are (``Device.load``, ``tensor_amd.torch.load``):

* ``rms_norm`` (``dtype``, ``residual``, ``out_dtype``, ``eps``): root-mean-square norm of rows, with the residual's addition;
* ``rms_norm_fp8`` (``dtype``, ``residual``, ``eps``): the same in 8 bits, a scale for each 128 columns of a row;
* ``quantize_fp8`` (``dtype``, ``gated``): rows, or silu(gate) * up of rows [gate | up], in 8 bits;
* ``fp8_linear`` (``out_dtype``): the linear layer on such rows and weights in 8 bits.

8 bits are e4m3 in ``uint8`` buffers (PyTorch's ``float8_e4m3fn``, viewed as ``uint8``).  The reference has no
counterpart: model inference is not part of it.
"""

from __future__ import annotations

import numpy as np

from tensor_amd.kernels.paged import _buffer, _fp32, _result as _manifest, _scalar

ENTRYPOINTS = {
    "rms_norm": "tensor_rms_norm_v1",
    "rms_norm_fp8": "tensor_rms_norm_fp8_v1",
    "quantize_fp8": "tensor_quantize_fp8_v1",
    "fp8_linear": "tensor_fp8_linear_v1",
}
DTYPES = ("float16", "float32")
BLOCK = 128            # columns of a row that share a scale, and rows of weights that do
LARGEST = 448.0        # of e4m3
SMALLEST_SCALE = 2.0 ** -126
NORM_MAX_WIDTH = 32768
NORM_LEAST_EPS = 2.0 ** -100


def _result(kernel: str, *arguments, **more) -> dict:
    return _manifest(kernel, *arguments, entrypoint=ENTRYPOINTS[kernel], **more)


def _blocks(name: str) -> dict:
    return {"op": "floordiv", "args": [{"op": "add", "args": [{"var": name}, BLOCK - 1]}, BLOCK]}


def _dtype(name: str, value) -> str:
    if str(value) not in DTYPES:
        raise ValueError(f"{name} must be one of {DTYPES}")
    return str(value)


def _norm(kernel: str, dtype, residual, out_dtype, eps) -> dict:
    dtype = _dtype("dtype", dtype)
    if residual is not None:
        residual = _dtype("residual", residual)
    if not NORM_LEAST_EPS <= _fp32(eps) < np.inf:
        raise ValueError("eps must be a finite number, 2^-100 at least")
    arguments = [_buffer("x", dtype, "M", "D")]
    if residual is not None:
        arguments.append(_buffer("residual", residual, "M", "D"))
    arguments.append(_buffer("weight", "float32", "D"))
    if out_dtype is None:
        arguments += [_buffer("codes", "uint8", "M", "D"), _buffer("scales", "float32", _blocks("D"), "M")]
        outputs = ["codes", "scales"]
    else:
        arguments.append(_buffer("out", out_dtype, "M", "D"))
        outputs = ["out"]
    if residual is not None:
        arguments.append(_buffer("residual_out", residual, "M", "D"))
        outputs.append("residual_out")
    label = ":".join([dtype, *([f"add:{residual}"] if residual else []), *([out_dtype] if out_dtype else []), str(float(eps))])
    return _result(kernel, label, [*arguments, _scalar("eps", "float32")], outputs, "M D", {"eps": float(eps)},
                   shape_domain={"D": [1, NORM_MAX_WIDTH]})


def norm_manifest(*, dtype="float16", residual=None, out_dtype="float16", eps: float = 1e-6) -> dict:
    """``residual``: None, or the type that the residual stream is held in (its sum is an output then)."""
    return _norm("rms_norm", dtype, residual, _dtype("out_dtype", out_dtype), eps)


def norm_fp8_manifest(*, dtype="float16", residual=None, eps: float = 1e-6) -> dict:
    return _norm("rms_norm_fp8", dtype, residual, None, eps)


def quantize_manifest(*, dtype="float16", gated: bool = False) -> dict:
    dtype = _dtype("dtype", dtype)
    if type(gated) is not bool:
        raise ValueError("gated must be a bool")
    if not gated:
        arguments = [_buffer("x", dtype, "M", "D"), _buffer("codes", "uint8", "M", "D"),
                     _buffer("scales", "float32", _blocks("D"), "M")]
        symbols, more = "M D", {}
    else:
        half = {"op": "floordiv", "args": [{"var": "G"}, 2]}
        blocks = {"op": "floordiv", "args": [{"op": "add", "args": [half, BLOCK - 1]}, BLOCK]}
        arguments = [_buffer("x", dtype, "M", "G"), _buffer("codes", "uint8", "M", half),
                     _buffer("scales", "float32", blocks, "M")]
        symbols, more = "M G", {"shape_divisors": {"G": 2}}
    return _result("quantize_fp8", dtype + (":gated" if gated else ""), [*arguments, _scalar("gated")], ["codes", "scales"],
                   symbols, {"gated": int(gated)}, **more)


def linear_manifest(*, out_dtype="float16") -> dict:
    out_dtype = _dtype("out_dtype", out_dtype)
    arguments = [
        _buffer("x", "uint8", "M", "K"), _buffer("x_scales", "float32", _blocks("K"), "M"),
        _buffer("w", "uint8", "N", "K"), _buffer("w_scales", "float32", _blocks("N"), _blocks("K")),
        _buffer("out", out_dtype, "M", "N"),
    ]
    return _result("fp8_linear", out_dtype, arguments, ["out"], "M N K", {}, shape_divisors={"K": 16},
                   shape_domain={"M": [1, 1 << 20], "N": [1, 1 << 22], "K": [1, 1 << 20]})


_MANIFESTS = {"rms_norm": norm_manifest, "rms_norm_fp8": norm_fp8_manifest, "quantize_fp8": quantize_manifest,
              "fp8_linear": linear_manifest}


def manifest(kernel: str, **options) -> dict:
    """The manifest of one norm or 8-bit operator with its options."""
    return _MANIFESTS[kernel](**options)


# ----------------------------------------------------------------- weights

def e4m3_values() -> np.ndarray:
    """The values of the 256 codes, fp32 (NaN at 0x7F and 0xFF)."""
    code = np.arange(256)
    exponent, fraction = (code >> 3) & 15, code & 7
    value = np.where(exponent == 0, fraction * 2.0 ** -9, (8 + fraction) * 2.0 ** (exponent - 10.0))
    value = np.where((code & 127) == 127, np.nan, value)
    return np.where(code >= 128, -value, value).astype(np.float32)


def e4m3_codes(values) -> np.ndarray:
    """The code nearest to each value (ties to the even one), uint8; past 448 the largest one, NaN where it is not finite."""
    values = np.asarray(values, np.float64)
    with np.errstate(invalid="ignore"):
        size = np.minimum(np.abs(np.where(np.isfinite(values), values, 0.0)), LARGEST)
        power = np.floor(np.log2(np.maximum(size, 2.0 ** -6)))
        steps = np.rint(size / 2.0 ** (power - 3))            # 8 to 16 of the power's eighths, or up to 8 below 2^-6
    code = np.where(size < 2.0 ** -6, steps, (power + 6) * 8 + steps).astype(np.int64)
    code = np.where(np.isfinite(values), code, 127)
    return (code + 128 * np.signbit(values)).astype(np.uint8)


def quantize_weight(weight) -> tuple:
    """(codes uint8 [N, K], scales fp32 [ceil(N / 128), ceil(K / 128)]) of a weight matrix, for ``fp8_linear``: each block's
    scale is its largest magnitude / 448 (2^-126 at least)."""
    weight = np.asarray(weight)
    if weight.ndim != 2 or not weight.size:
        raise ValueError("a weight matrix has two dimensions")
    if np.iscomplexobj(weight):
        raise ValueError("weights must be real numbers")
    if not np.isfinite(weight).all():
        raise ValueError("weights must be finite")
    if max(-float(weight.min()), float(weight.max())) / LARGEST > float(np.finfo(np.float32).max):
        raise ValueError("weights of these magnitudes have no scale in fp32")
    rows, columns = weight.shape
    codes = np.empty(weight.shape, np.uint8)
    scales = np.empty((-(-rows // BLOCK), -(-columns // BLOCK)), np.float32)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = np.s_[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK]
            block = weight[at].astype(np.float64)
            scales[i, j] = max(np.abs(block).max() / LARGEST, SMALLEST_SCALE)
            codes[at] = e4m3_codes(block / float(scales[i, j]))
    return codes, scales
