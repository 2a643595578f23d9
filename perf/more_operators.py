"""Representative calls of the norm and 8-bit operators, and how to time and check one.

They are what a decoder layer runs around its attention when its linears are held in 8 bits (e4m3, a scale
for each block of 128):

* ``norm`` (``rms_norm``): root-mean-square norm of rows, with the residual's addition or without.
* ``norm_fp8`` (``rms_norm_fp8``): the same, its result in 8 bits with a scale for each 128 columns of a row.
* ``quantize`` (``quantize_fp8``): rows, or silu(gate) * up of rows [gate | up], in 8 bits with scales.
* ``linear`` (``fp8_linear``): the product of such rows with a weight matrix in 8 bits, a scale for each of its
  128 x 128 blocks.

Scales of rows are held [blocks, rows].  Sizes, types and layouts are the case's; the seed makes the values.
"""

from __future__ import annotations

import functools
import math

import torch

own = False

BLOCK = 128
LARGEST = 448.0          # of e4m3
SMALLEST = 2.0 ** -126   # a scale
EPS = 1e-6

# ------------------------------------------------------------------- cases


def _norm(name, op, rows, width, dtype, residual, out="float16"):
    """residual: "none", or the type that the residual stream is held in."""
    case = {"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype, "residual": residual}
    if op == "norm":
        case["out"] = out
    return case


def _quantize(name, rows, width, dtype, gated):
    return {"name": name, "op": "quantize", "rows": rows, "width": width, "dtype": dtype, "gated": gated}


def _linear(name, m, n, k, out):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "out": out}


def listed():
    return [
        # before the last linear of a decode step, one sequence: latency only
        _norm("norm_t1_add", "norm", 1, 4096, "float16", "float16"),
        # the norm of each head of a prompt's queries and keys: very many short rows
        _norm("norm_heads_d128", "norm", 81880, 128, "float16", "none"),
        # before a layer's linears, a decode step of 64 sequences, the residual stream in 32 bits
        _norm("norm_fp8_t64_add32", "norm_fp8", 64, 4096, "float16", "float32"),
        # the same of a long prompt
        _norm("norm_fp8_t8192_add", "norm_fp8", 8192, 4096, "float16", "float16"),
        # attention's output of a few sequences before the output linear
        _quantize("quantize_t8", 8, 4096, "float16", False),
        # a prompt's gate and up rows before the down linear
        _quantize("quantize_t4093_gated", 4093, 12288, "float16", True),
        # one token through gate + up of a decode step: the weights' bytes
        _linear("linear_m1_gate_up", 1, 24576, 4096, "float16"),
        # sixteen sequences through the down linear: long rows, few outputs
        _linear("linear_m16_down", 16, 4096, 12288, "float16"),
        # a ragged batch through a smaller layer, sizes that end inside tiles and blocks, fp32 outputs
        _linear("linear_m77_ragged", 77, 2500, 2544, "float32"),
        # a prompt chunk through q + k + v
        _linear("linear_m333_qkv", 333, 6144, 4096, "float16"),
        # a prompt through the output linear
        _linear("linear_m2048_o", 2048, 4096, 4096, "float16"),
        # a long prompt through gate + up: the most arithmetic of one call
        _linear("linear_m8192_gate_up", 8192, 24576, 4096, "float16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "norm_fp8", "quantize", "linear", "linear", "linear"))
    if op in ("norm", "norm_fp8"):
        width = rng.choice((128, 2560, 4096, 5120, 8192, 16 * _log_int(rng, 4, 1024), _log_int(rng, 64, 16384)))
        case = _norm("", op, max(1, min(_log_int(rng, 1, 65536), 8192 * 4096 // width)), width,
                     rng.choice(("float16", "float16", "float32")), rng.choice(("none", "float16", "float32")),
                     rng.choice(("float16", "float16", "float32")))
    elif op == "quantize":
        width = rng.choice((2560, 4096, 12288, 16 * _log_int(rng, 8, 1024), _log_int(rng, 64, 16384)))
        case = _quantize("", max(1, min(_log_int(rng, 1, 16384), 4096 * 12288 // width)), width,
                         rng.choice(("float16", "float16", "float32")), rng.random() < 0.5)
    else:
        m = _log_int(rng, 1, rng.choice((16, 256, 8192)))
        case = _linear("", m, _log_int(rng, 64, 24576), 16 * _log_int(rng, 8, 768), rng.choice(("float16", "float16", "float32")))
        while 2 * m * case["n"] * case["k"] > 2 * 8192 * 24576 * 4096:
            case["n"] = case["n"] * 3 // 4
    del case["name"]
    return case


def _blocks(n):
    return -(-n // BLOCK)


def _size(dtype):
    return 2 if dtype == "float16" else 4


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * _blocks(k) * (m + _blocks(n)) + _size(case["out"]) * m * n, "flops": 2 * m * n * k}
    rows, width = case["rows"], case["width"]
    if case["op"] == "quantize":
        return {"bytes": rows * width * (_size(case["dtype"]) * (2 if case["gated"] else 1) + 1) + 4 * rows * _blocks(width),
                "flops": rows * width * (8 if case["gated"] else 3)}
    result = _size(case["out"]) * rows * width if case["op"] == "norm" else rows * width + 4 * rows * _blocks(width)
    stream = 0 if case["residual"] == "none" else 2 * _size(case["residual"])
    return {"bytes": rows * width * (_size(case["dtype"]) + stream) + 4 * width + result,
            "flops": rows * width * (5 if case["op"] == "norm" else 8)}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    return generator


def _normal(generator, shape, scale=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=generator)


def _uniform(generator, shape, low, high):
    return torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(low, high, generator=generator)


def _outliers(generator, width):
    """What activations are like: a few columns are an order of magnitude larger than the others."""
    return 1.0 + 20.0 * (_uniform(generator, (width,), 0.0, 1.0) > 0.995)


def _inputs(case, seed):
    g = _generator(seed)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x, x_scales = _in_8_bits(_normal(g, (m, k)) * _outliers(g, k))
        w = _normal(g, (n, k), k ** -0.5)
        spread = _uniform(g, (_blocks(n), _blocks(k)), 0.5, 2.0)
        wide = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK)).view(_blocks(n), BLOCK, _blocks(k), BLOCK)
        wide = wide * spread[:, None, :, None]
        w_scales = wide.abs().amax((1, 3)) / LARGEST
        codes = (wide / w_scales[:, None, :, None]).view(-1, wide.shape[2] * BLOCK)[:n, :k].to(torch.float8_e4m3fn)
        return {"x": x.view(torch.uint8), "x_scales": x_scales, "w": codes.contiguous().view(torch.uint8), "w_scales": w_scales}
    dtype, rows, width = getattr(torch, case["dtype"]), case["rows"], case["width"]
    if case["op"] == "quantize":
        if case["gated"]:  # the gate rows, then the up rows
            return {"x": (_normal(g, (rows, 2 * width), 1.5) * torch.cat([torch.ones(width, device="cuda"),
                                                                         _outliers(g, width)])).to(dtype)}
        return {"x": (_normal(g, (rows, width)) * _outliers(g, width)).to(dtype)}
    state = {"x": (_normal(g, (rows, width)) * _outliers(g, width)).to(dtype), "weight": _uniform(g, (width,), 0.2, 1.8)}
    if case["residual"] != "none":
        state["r"] = (_normal(g, (rows, width), 4.0) * _outliers(g, width)).to(getattr(torch, case["residual"]))
    return state


@functools.lru_cache(maxsize=None)
def _kernel(name, **options):
    import tensor_amd.torch as tt

    return tt.load(name, **options)


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if not own:
        return state
    if case["op"] == "linear":
        kernel, names = _kernel("fp8_linear", out_dtype=case["out"]), ("x", "x_scales", "w", "w_scales")
    elif case["op"] == "quantize":
        kernel, names = _kernel("quantize_fp8", dtype=case["dtype"], gated=case["gated"]), ("x",)
    else:
        residual = None if case["residual"] == "none" else case["residual"]
        options = dict(dtype=case["dtype"], residual=residual, eps=EPS)
        kernel = _kernel("rms_norm_fp8", **options) if case["op"] == "norm_fp8" else _kernel(
            "rms_norm", out_dtype=case["out"], **options)
        names = ("x", "r", "weight") if residual else ("x", "weight")
    state["call"] = kernel.prepare(*(state[name] for name in names))
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        state["call"]()
        outputs = state["call"].outputs
        return outputs if op in ("norm", "linear") else (outputs[0].view(torch.float8_e4m3fn), *outputs[1:])
    return {"norm": _plain_norm, "norm_fp8": _plain_norm, "quantize": _plain_quantize, "linear": _plain_linear}[op](state)


# ------------------------------------------------------------- plain forms


def _in_8_bits(y):
    """(codes [rows, width], scales [blocks, rows]) of rows in fp32."""
    rows, width = y.shape
    blocks = torch.nn.functional.pad(y, (0, -width % BLOCK)).view(rows, -1, BLOCK)
    scales = (blocks.abs().amax(-1) / LARGEST).clamp_min(SMALLEST)
    codes = (blocks / scales[..., None]).to(torch.float8_e4m3fn)
    return codes.view(rows, -1)[:, :width].contiguous(), scales.t().contiguous()


def _plain_norm(state):
    case, h = state["case"], state["x"].float()
    if case["residual"] != "none":
        h = h + state["r"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * state["weight"]
    result = (y.to(getattr(torch, case["out"])),) if case["op"] == "norm" else _in_8_bits(y)
    return result if case["residual"] == "none" else (*result, h.to(state["r"].dtype))


def _plain_quantize(state):
    y = state["x"].float()
    if state["case"]["gated"]:
        gate, up = y.chunk(2, -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return _in_8_bits(y)


def _plain_linear(state):
    n, k = state["w"].shape
    x = state["x"].view(torch.float8_e4m3fn).float() * state["x_scales"].t().repeat_interleave(BLOCK, 1)[:, :k]
    scales = state["w_scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    w = state["w"].view(torch.float8_e4m3fn).float() * scales
    return (torch.mm(x, w.t()).to(getattr(torch, state["case"]["out"])),)


# ------------------------------------------------------- the same in 64 bits


def _nearest_e4m3(v):
    """The e4m3 value nearest to each of v, ties to the even one: steps of 2^-3 of the power of two below, 2^-9 at least."""
    power = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(power - 3.0)
    return (torch.round(v / step) * step).clamp(-LARGEST, LARGEST)


def _blocks_of(y):
    """Values of [rows, width] in 64 bits as e4m3 gives them, and their scales, a block of columns at a time."""
    values, scales = torch.empty_like(y), []
    for first in range(0, y.shape[1], BLOCK):
        part = y[:, first:first + BLOCK]
        scale = torch.clamp(torch.linalg.vector_norm(part, ord=math.inf, dim=1) / LARGEST, min=SMALLEST)
        values[:, first:first + BLOCK] = _nearest_e4m3(part / scale[:, None])
        scales.append(scale)
    return values, torch.stack(scales)


def _value(codes):
    """The e4m3 values of bytes: sign, four bits of exponent (bias 7), three of fraction."""
    byte = torch.arange(256, device="cuda")
    exponent, fraction = (byte >> 3) & 15, (byte & 7).double()
    value = torch.where(exponent == 0, fraction * 2.0 ** -9, (8.0 + fraction) * torch.exp2(exponent.double() - 10.0))
    value = torch.where((byte & 127) == 127, torch.full_like(value, math.nan), value)
    return torch.where(byte >= 128, -value, value)[codes.long()]


def exact(case, seed):
    inputs = _inputs(case, seed)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        out = torch.zeros((m, n), dtype=torch.float64, device="cuda")
        for first in range(0, n, 8 * BLOCK):  # eight blocks of weight rows at a time
            w = _value(inputs["w"][first:first + 8 * BLOCK])
            for row in range(0, w.shape[0], BLOCK):
                for b in range(_blocks(k)):
                    w[row:row + BLOCK, b * BLOCK:(b + 1) * BLOCK] *= inputs["w_scales"][(first + row) // BLOCK, b].double()
            for top in range(0, m, 2048):
                x = _value(inputs["x"][top:top + 2048])
                for b in range(_blocks(k)):
                    x[:, b * BLOCK:(b + 1) * BLOCK] *= inputs["x_scales"][b, top:top + 2048, None].double()
                out[top:top + 2048, first:first + 8 * BLOCK] = x @ w.T
        return (out,)
    x = inputs["x"].double()
    if case["op"] == "quantize":
        if case["gated"]:
            gate, up = x[:, :case["width"]], x[:, case["width"]:]
            x = gate * torch.sigmoid(gate) * up
        return _blocks_of(x)
    total = x if case["residual"] == "none" else x + inputs["r"].double()
    length = torch.linalg.vector_norm(total, dim=1, keepdim=True)
    y = total / torch.sqrt(length ** 2 / case["width"] + EPS) * inputs["weight"].double()
    result = (y,) if case["op"] == "norm" else _blocks_of(y)
    return result if case["residual"] == "none" else (*result, total)
