"""Manifests of the paged-cache operators (include/tensor_hip.h) and the rotary angle table.

They stand between a layer's q + k + v linears and its output linear and are loaded by name as the
GGUF kernels are (``Device.load``, ``tensor_amd.torch.load``):

* ``paged_slots`` (``page_size``): a step's block tables, slots and positions from request lengths;
* ``rotary`` (``layout``, ``dtype``, ``inverse``): rotary positions of queries and keys, or their gradient;
* ``rotary_store`` (``layout``, ``dtype``): the same, keys and values written to their cache slots;
* ``paged_attention`` (``scale``): attention over a shared prefix and each request's own pages.

The reference has no counterpart: model inference is not part of it.
"""

from __future__ import annotations

import math

import numpy as np

ENTRYPOINTS = {
    "paged_slots": "tensor_paged_slots_v1",
    "rotary": "tensor_rotary_v1",
    "rotary_store": "tensor_rotary_store_v1",
    "paged_attention": "tensor_paged_attention_v1",
}
LAYOUTS = ("half", "interleaved")  # pairs (p, p + rotated / 2), pairs (2 p, 2 p + 1)
DTYPES = ("float16", "float32")
HEAD_DIMS = (64, 128)   # of paged_attention
MAX_REQUESTS = 1024     # of paged_attention
MAX_PAGE_SIZE = 1024    # pages hold a power of two of tokens


def _buffer(name: str, dtype: str, *shape, alignment: int | None = None) -> dict:
    return {"name": name, "dtype": dtype, "shape": [{"var": extent} if isinstance(extent, str) else extent for extent in shape],
            "alignment": alignment or (4 if dtype == "int32" else 16)}


def _scalar(name: str, dtype: str = "uint32") -> dict:
    return {"name": name, "dtype": dtype, "kind": "scalar"}


def _result(kernel: str, label: str, arguments: list, outputs: list, symbols: str, constants: dict, *,
            entrypoint: str | None = None, **more) -> dict:
    return {
        "name": f"{kernel}:{label}",
        "provider": "hip",
        "target": "gfx950",
        "entrypoint": entrypoint or ENTRYPOINTS[kernel],
        "runtime_abi": {"major": 1, "minor": 1, "required_capabilities": [
            "contiguous", "executable_descriptors", "no_external_workspace", "scalars"]},
        "arguments": arguments,
        "abi": [dict(item, kind=item.get("kind", "buffer")) for item in arguments],
        "outputs": outputs,
        "constants": constants,
        "symbols": {name: "int32" for name in symbols.split()},
        # the entry point chooses its own launch geometry
        "launch": {"grid": [1, 1, 1], "block": [256, 1, 1], "shared_memory_bytes": 0},
        **more,
    }


def slots_manifest(*, page_size: int) -> dict:
    if type(page_size) is not int or not 1 <= page_size <= MAX_PAGE_SIZE or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 1 to {MAX_PAGE_SIZE}")
    arguments = [
        _buffer("lengths", "int32", "B"), _buffer("counts", "int32", "B"), _buffer("start", "int32", 1),
        _buffer("free", "int32", "F"), _buffer("free_count", "int32", 1), _buffer("table", "int32", "B", "P"),
        _scalar("T", "int32"),
        _buffer("offsets", "int32", {"op": "add", "args": [{"var": "B"}, 1]}), _buffer("lengths_out", "int32", "B"),
        _buffer("positions", "int32", "T"), _buffer("slots", "int32", "T"), _buffer("table_out", "int32", "B", "P"),
        _buffer("free_left", "int32", 1), _scalar("page_size"),
    ]
    return _result("paged_slots", str(page_size), arguments,
                   ["offsets", "lengths_out", "positions", "slots", "table_out", "free_left"], "B F P T",
                   {"page_size": page_size}, shape_domain={"T": [1, (1 << 31) - 1]})


def _rotary_options(layout: str, dtype) -> tuple:
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}")
    if str(dtype) not in DTYPES:
        raise ValueError(f"dtype must be one of {DTYPES}")
    return LAYOUTS.index(layout), str(dtype)


def rotary_manifest(*, layout: str = "half", dtype="float16", inverse: bool = False) -> dict:
    code, dtype = _rotary_options(layout, dtype)
    if type(inverse) is not bool:
        raise ValueError("inverse must be a bool")
    arguments = [
        _buffer("q", dtype, "T", "H", "D"), _buffer("k", dtype, "T", "G", "D"), _buffer("positions", "int32", "T"),
        _buffer("angles", "float32", "S", "R"), _buffer("q_out", dtype, "T", "H", "D"),
        _buffer("k_out", dtype, "T", "G", "D"), _scalar("layout"), _scalar("inverse"),
    ]
    return _result("rotary", f"{layout}:{dtype}" + (":inverse" if inverse else ""), arguments, ["q_out", "k_out"],
                   "T H G D S R", {"layout": code, "inverse": int(inverse)}, shape_divisors={"R": 2})


def rotary_store_manifest(*, layout: str = "half", dtype="float16") -> dict:
    code, dtype = _rotary_options(layout, dtype)
    cache = ("N", "G", "L", "D")
    arguments = [
        _buffer("q", dtype, "T", "H", "D"), _buffer("k", dtype, "T", "G", "D"), _buffer("v", dtype, "T", "G", "D"),
        _buffer("positions", "int32", "T"), _buffer("slots", "int32", "T"), _buffer("angles", "float32", "S", "R"),
        _buffer("q_out", "float16", "T", "H", "D"), _buffer("k_cache", "float16", *cache),
        _buffer("v_cache", "float16", *cache), _scalar("layout"),
    ]
    # no declared outputs: the caches are updated in place, so every buffer is the caller's
    return _result("rotary_store", f"{layout}:{dtype}", arguments, [], "T H G D S R N L", {"layout": code},
                   shape_divisors={"R": 2}, mutable_inputs=["q_out", "k_cache", "v_cache"])


def _fp32(value) -> float:
    """A number as fp32 holds it, infinite past its largest; NaN for what is no number."""
    if not isinstance(value, (int, float)) or isinstance(value, bool):
        return math.nan
    try:
        with np.errstate(over="ignore"):
            return float(np.float32(value))
    except OverflowError:  # whole numbers past 64-bit floats
        return math.copysign(math.inf, 1 if value > 0 else -1)


def attention_manifest(*, scale: float | None = None) -> dict:
    if scale is not None and not 0.0 < _fp32(scale) < math.inf:
        raise ValueError("scale must be a positive finite number")
    cache = ("N", "G", "L", "D")
    arguments = [
        _buffer("q", "float16", "T", "H", "D"), _buffer("k_cache", "float16", *cache),
        _buffer("v_cache", "float16", *cache), _buffer("offsets", "int32", {"op": "add", "args": [{"var": "B"}, 1]}),
        _buffer("lengths", "int32", "B"), _buffer("table", "int32", "B", "P"), _buffer("prefix_pages", "int32", "PP"),
        _buffer("prefix_length", "int32", 1), _buffer("workspace", "uint8", "W", alignment=256),
        _buffer("out", "float16", "T", "H", "D"), _scalar("scale", "float32"),
    ]
    return _result("paged_attention", "default" if scale is None else str(float(scale)), arguments, ["out"],
                   "T H G D N L B P PP W", {"scale": 0.0 if scale is None else float(scale)},
                   shape_domain={"D": [min(HEAD_DIMS), max(HEAD_DIMS)], "B": [1, MAX_REQUESTS]},
                   shape_divisors={"D": 64}, scratch=["workspace"])


_MANIFESTS = {"paged_slots": slots_manifest, "rotary": rotary_manifest, "rotary_store": rotary_store_manifest,
              "paged_attention": attention_manifest}


def manifest(kernel: str, **options) -> dict:
    """The manifest of one paged-cache operator with its options."""
    return _MANIFESTS[kernel](**options)


# ------------------------------------------------------------------ angles

def rotary_angles(reach: int, rotated: int, *, base: float = 10000.0, scaling: str | None = None,
                  factor: float = 1.0, original: int | None = None, fast: float = 32.0,
                  slow: float = 1.0) -> np.ndarray:
    """The angle table of ``rotary`` and ``rotary_store``: fp32 [reach, rotated], the cosines of the
    rotated / 2 pairs at each position, then their sines, computed in 64 bits and rounded once.

    Pair p turns by ``base ** (-2 p / rotated)`` a position.  For contexts ``factor`` times the trained
    length, ``scaling`` is one of

    * ``linear``: positions divided by the factor;
    * ``ntk``: the base raised so that the slowest pair is slowed by the factor and the fastest kept;
    * ``yarn``: pairs that turn more than ``fast`` times in ``original`` positions kept, those that turn less
      than ``slow`` times slowed by the factor, a ramp over the pairs between, and cosines and sines scaled by
      f = 0.1 ln(factor) + 1 (``rotary`` with ``inverse`` after ``rotary`` gives f^2 times its input then).
    """
    if type(reach) is not int or type(rotated) is not int or reach < 1 or rotated < 2 or rotated % 2:
        raise ValueError("reach must be a positive integer and rotated a positive even one")
    if not (math.isfinite(base) and base > 1.0) or not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    if scaling is None and factor != 1.0:
        raise ValueError("factor needs a scaling")
    if scaling == "ntk":
        if rotated < 4:
            raise ValueError("ntk scaling needs two pairs")
        base = base * factor ** (rotated / (rotated - 2))
    pair = np.arange(rotated // 2, dtype=np.float64)
    frequency = base ** (-2.0 * pair / rotated)
    magnitude = 1.0
    if scaling == "linear":
        frequency = frequency / factor
    elif scaling == "yarn":
        if type(original) is not int or original < 1 or not 0.0 < slow < fast:
            raise ValueError("yarn scaling needs the original length and 0 < slow < fast")

        def pair_of(turns: float) -> float:  # the pair that makes so many turns in the original length
            return rotated * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

        low = max(math.floor(pair_of(fast)), 0)
        high = min(math.ceil(pair_of(slow)), rotated - 1)
        ramp = np.clip((pair - low) / max(high - low, 1e-3), 0.0, 1.0)
        frequency = frequency / factor * ramp + frequency * (1.0 - ramp)
        magnitude = 0.1 * math.log(factor) + 1.0
    angle = np.arange(reach, dtype=np.float64)[:, None] * frequency
    return (magnitude * np.concatenate([np.cos(angle), np.sin(angle)], axis=1)).astype(np.float32)
