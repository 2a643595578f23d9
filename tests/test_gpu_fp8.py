"""The norm and the 8-bit operators on a GPU against their plain forms in 64 bits (tests/fp8_cases.py)."""

from __future__ import annotations

import numpy as np
import pytest

from tests import fp8_cases as plain
from tests.test_gpu_paged import Buffers

pytestmark = pytest.mark.gpu

WIDTHS = [1, 3, 7, 8, 9, 16, 100, 127, 128, 129, 136, 250, 512, 520, 1000, 2048, 2051, 2560, 4096, 4104, 5120, 8192, 8200,
          12289, 16384, 16390, 32768]


def run_norm(device, x, residual, weight, eps, out):
    """[y, (h)] or [codes, scales, (h)] for out = "codes"."""
    codes = out == "codes"
    options = dict(dtype=str(x.dtype), residual=None if residual is None else str(residual.dtype), eps=eps)
    if not codes:
        options["out_dtype"] = out
    with Buffers(device) as put:
        kernel = device.load("rms_norm_fp8" if codes else "rms_norm", **options)
        rows, width = x.shape
        outs = [put.empty((rows, width), "uint8"), put.empty((plain.blocks_of(width), rows), "float32")] if codes else [
            put.empty((rows, width), out)]
        inputs = [put(x)]
        if residual is not None:
            inputs.append(put(residual))
            outs.append(put.empty((rows, width), str(residual.dtype)))
        kernel.launch(*inputs, put(weight), *outs)
        return [o.to_numpy() for o in outs]


def check_norm(device, x, residual, weight, eps, out):
    got = run_norm(device, x, residual, weight, eps, out)
    want, h = plain.norm(x, residual, weight, eps)
    if residual is not None:
        plain.check_rounded(got.pop(), h, str(residual.dtype), 2.0 ** -24)
    if out == "codes":
        plain.check_codes(*got, want, plain.NORM_OFF)
    else:
        plain.check_rounded(got[0], want, out, plain.NORM_OFF)


@pytest.mark.parametrize("out", ["float16", "float32", "codes"])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(hip_device, width, out):
    rng = np.random.default_rng(width)
    weight = rng.uniform(-1, 2, width).astype(np.float32)
    for rows, dtype, residual in ((1, "float16", None), (5, "float16", "float16"), (35, "float16", "float32"),
                                  (3, "float32", "float32"), (2, "float32", None), (17, "float32", "float16")):
        x = (3 * rng.standard_normal((rows, width))).astype(dtype)
        r = None if residual is None else (5 * rng.standard_normal((rows, width))).astype(residual)
        print(f"[case] norm {rows} x {width} {dtype} {residual} {out}", flush=True)
        check_norm(hip_device, x, r, weight, 1e-6, out)


@pytest.mark.parametrize("out", ["float16", "float32", "codes"])
@pytest.mark.parametrize("width", [5, 128, 300, 4096, 9000])
def test_norm_of_small_large_and_other_values(hip_device, width, out):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((9, width)).astype(np.float32)
    weight = rng.uniform(0.5, 1.5, width).astype(np.float32)
    x[0] = 0.0
    x[1] *= 1e-20     # squares below fp32: eps alone
    x[2] *= 1e25      # squares past fp32
    x[3] *= 1e38 / np.abs(x[3]).max() * 3
    x[4, -1] = np.nan
    x[6, 0] = 1e30    # one value outweighs the others
    for eps in (1e-6, 1e-12, 0.5):
        check_norm(hip_device, x, None, weight, eps, out)
    x[5, 0] = np.inf  # infinity / infinity there, 0 elsewhere
    got = run_norm(hip_device, x, None, weight, 1e-6, out)
    row = plain.value(got[0])[5] if out == "codes" else got[0][5]
    assert np.isnan(row[0]) and (row[1:] == 0).all()
    assert np.isnan(plain.value(got[0])[4] if out == "codes" else got[0][4]).all()


@pytest.mark.parametrize("width", [1, 5, 300, 9000])
def test_norm_of_the_largest_and_least_eps(hip_device, width):
    """Beside squares whose sum passes fp32, and beside such as are lost below it."""
    rng = np.random.default_rng(width)
    weight = np.ones(width, np.float32)
    for size, eps in ((1e19, 1e38), (1e19, 1e36), (1.5e19, 3e38), (1e18, 3e38), (1e-15, 2.0 ** -100), (1e-25, 2.0 ** -100)):
        x = (size * rng.uniform(0.8, 1.2, (3, width))).astype(np.float32)
        check_norm(hip_device, x, None, weight, eps, "float32")


def test_norm_sums_are_not_rounded_before_the_norm(hip_device):
    """Sums next to each other in fp16 differ in the result: h enters in fp32."""
    x = np.full((1, 128), 2048, np.float16)
    r = np.linspace(0, 1, 128).astype(np.float16)[None]
    y, h = run_norm(hip_device, x, r, np.ones(128, np.float32), 1e-6, "float32")
    want, sums = plain.norm(x, r, np.ones(128), 1e-6)
    assert (np.abs(y - want) <= plain.NORM_OFF * want + 2.0 ** -24).all() and len(np.unique(y)) > 100
    assert np.array_equal(h, sums.astype(np.float32).astype(np.float16))


@pytest.mark.parametrize("width", [100, 128, 130, 4096, 6000, 20000])
def test_norm_in_place(hip_device, width):
    rng = np.random.default_rng(width)
    x, r = (rng.standard_normal((37, width)).astype(np.float16) for _ in range(2))
    weight = rng.uniform(0.5, 1.5, width).astype(np.float32)
    want = run_norm(hip_device, x, r, weight, 1e-5, "float16")
    with Buffers(hip_device) as put:
        kernel = hip_device.load("rms_norm", residual="float16", eps=1e-5)
        xb, rb = put(x), put(r)
        kernel.launch(xb, rb, put(weight), xb, rb)
        assert np.array_equal(xb.to_numpy(), want[0]) and np.array_equal(rb.to_numpy(), want[1])


@pytest.mark.parametrize("out", ["float16", "float32", "codes"])
@pytest.mark.parametrize("width", [2049, 2560, 4096, 4100, 5120, 6144, 6150, 8192])
def test_norm_of_rows_past_the_few(hip_device, width, out):
    """512 rows are shared by more threads each than 513."""
    rng = np.random.default_rng(width)
    weight = rng.uniform(-1, 2, width).astype(np.float32)
    for rows, dtype, residual in ((512, "float16", "float16"), (513, "float16", "float32"), (513, "float32", None)):
        x = (3 * rng.standard_normal((rows, width))).astype(dtype)
        r = None if residual is None else (5 * rng.standard_normal((rows, width))).astype(residual)
        x[rows // 2] *= 1e25 if dtype == "float32" else 0  # squares past fp32, or the residual's alone
        print(f"[case] norm {rows} x {width} {dtype} {residual} {out}", flush=True)
        check_norm(hip_device, x, r, weight, 1e-6, out)


def test_norm_of_many_rows(hip_device):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((70001, 64)).astype(np.float16)
    check_norm(hip_device, x, None, np.ones(64, np.float32), 1e-6, "codes")


# ---------------------------------------------------------------- quantize

def run_quantize(device, x, gated=False):
    with Buffers(device) as put:
        rows, width = x.shape[0], x.shape[1] // (2 if gated else 1)
        outs = put.empty((rows, width), "uint8"), put.empty((plain.blocks_of(width), rows), "float32")
        device.load("quantize_fp8", dtype=str(x.dtype), gated=gated).launch(put(x), *outs)
        return [o.to_numpy() for o in outs]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize(hip_device, width, dtype):
    rng = np.random.default_rng(width)
    for rows in (1, 33, 67):
        x = (np.exp(2 * rng.standard_normal((rows, 1))) * rng.standard_normal((rows, 2 * width))).astype(dtype)
        print(f"[case] quantize {rows} x {width} {dtype}", flush=True)
        plain.check_codes(*run_quantize(hip_device, x[:, :width].copy()), x[:, :width].astype(np.float64), 0.0)
        # exp of up to 6 sigma and more: its argument is rounded twice, 2^-23 of it, and it is within 2^-22; the sum, the
        # quotient and the product add 2^-22
        off = 2.0 ** -21 + 2.0 ** -23 * float(np.abs(x).max())
        plain.check_codes(*run_quantize(hip_device, x, True), plain.gated(x), off)


def test_quantize_other_values(hip_device):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((8, 300)).astype(np.float32)
    x[0] = 0.0
    x[1] *= 1e-41        # below the smallest scale
    x[2] *= 1e37
    x[3, 5] = np.inf
    x[3, 130] = -np.inf
    x[4, 299] = np.nan
    x[5, :128] = np.nan  # nothing finite in a block
    x[6, 0] = 3.4e38
    plain.check_codes(*run_quantize(hip_device, x), x.astype(np.float64), 0.0)
    # every code from the value that it stands for, and ties
    values = plain.value(np.array([c for c in range(127)]))
    ties = (values[1:] + values[:-1]) / 2
    row = np.concatenate([values, [448.0], ties, [0.0, 448.0]])
    codes, scales = run_quantize(hip_device, row[None].astype(np.float32))
    assert (scales == 1.0).all()
    assert np.array_equal(codes[0][:127], np.arange(127))
    assert np.array_equal(codes[0][128:254], np.where(np.arange(126) % 2, np.arange(1, 127), np.arange(126)))


def test_gated_far_gates(hip_device):
    """Gates far below zero close, far above pass; exp of neither end harms."""
    g = np.array([-65504, -1000, -100, -89, -50, 0, 50, 89, 100, 1000, 60000], np.float16)
    x = np.concatenate([g, np.ones_like(g)])[None]
    codes, scales = run_quantize(hip_device, x, True)
    plain.check_codes(codes, scales, plain.gated(x), 2.0 ** -14)
    assert (codes[0, :4] & 127 == 0).all()
    # alone in its block a closed gate's value is what there is: down to the smallest scale and past it
    for g, v in ((-79.5, 3.0), (-80.5, 3.0), (-88.0, -7.0), (-95.0, 2000.0), (-120.0, 60000.0), (-104.0, 1.0), (-60000.0, 60000.0)):
        x = np.array([[g, v]], np.float16)
        plain.check_codes(*run_quantize(hip_device, x, True), plain.gated(x), 2.0 ** -14)
    x = np.array([[-150.0, 3e38], [-200.0, -1e30], [-700.0, 3e38], [-3e38, 3e38]], np.float32)
    plain.check_codes(*run_quantize(hip_device, x, True), plain.gated(x), 2.0 ** -12)


# ------------------------------------------------------------------ linear

def run_linear(device, x, x_scales, w, w_scales, out_dtype):
    with Buffers(device) as put:
        out = put.empty((x.shape[0], w.shape[0]), out_dtype)
        device.load("fp8_linear", out_dtype=out_dtype).launch(put(x), put(x_scales), put(w), put(w_scales), out)
        return out.to_numpy()


def operands(seed, m, n, k):
    rng = np.random.default_rng(seed)
    x_scales = np.exp2(rng.uniform(-12, 2, (plain.blocks_of(k), m))).astype(np.float32)
    w_scales = np.exp2(rng.uniform(-16, -8, (plain.blocks_of(n), plain.blocks_of(k)))).astype(np.float32)
    return plain.random_codes(rng, (m, k)), x_scales, plain.random_codes(rng, (n, k)), w_scales


SHAPES = [(m, n, k) for m, n, k in (
    (1, 1, 16), (1, 17, 128), (2, 300, 144), (3, 16, 4112), (1, 513, 1040), (8, 129, 2064), (15, 100, 112), (16, 16, 256),
    (17, 40, 272), (31, 257, 1040), (33, 384, 384), (48, 65, 16), (63, 640, 1168), (64, 64, 12288), (65, 130, 896),
    (77, 250, 2544), (96, 33, 528), (127, 129, 128), (128, 128, 128), (129, 127, 1296), (200, 700, 640), (255, 255, 272),
    (256, 256, 256), (257, 300, 1040), (300, 1100, 400), (511, 260, 144), (700, 900, 80), (1025, 520, 528), (1, 9000, 256),
    (40, 4100, 272), (130, 8200, 144), (700, 6200, 1040), (4000, 4090, 1040))]  # the last ones: of each tile many


@pytest.mark.parametrize("out_dtype", ["float16", "float32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear(hip_device, shape, out_dtype):
    print(f"[case] linear {shape} {out_dtype}", flush=True)
    call = operands(sum(shape), *shape)
    got = run_linear(hip_device, *call, out_dtype)
    if shape[0] > 512:  # some rows of large calls: the first and last ones, others at random
        rows = np.unique(np.concatenate([np.arange(20), np.arange(shape[0] - 20, shape[0]),
                                         np.random.default_rng(1).integers(0, shape[0], 60)]))
        call, got = (call[0][rows], np.ascontiguousarray(call[1][:, rows]), *call[2:]), got[rows]
    cut = plain.cut_off(*call) if out_dtype == "float16" else 0.0
    plain.check_linear(got, *plain.linear(*call), shape[2], cut)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_of_whole_numbers_is_exact(hip_device, shape):
    """Small whole numbers and scales that are powers of two: every sum is a whole number of 2^-6 below 2^18, so fp32 holds
    each on the way, whatever the order, and a value lost, doubled or from elsewhere shows."""
    m, n, k = shape
    rng = np.random.default_rng(7)
    codes = np.array([0x00, 0x38, 0x40, 0x44, 0xB8, 0xC0, 0xC4], np.uint8)  # 0, 1, 2, 3 and their negatives
    x, w = codes[rng.integers(0, 7, (m, k))], codes[rng.integers(0, 7, (n, k))]
    x_scales = np.exp2(rng.integers(-3, 1, (plain.blocks_of(k), m))).astype(np.float32)
    w_scales = np.exp2(rng.integers(-3, 1, (plain.blocks_of(n), plain.blocks_of(k)))).astype(np.float32)
    want, size = plain.linear(x, x_scales, w, w_scales)
    assert size.max() < 2.0 ** 18
    got = run_linear(hip_device, x, x_scales, w, w_scales, "float32")
    assert np.array_equal(got.astype(np.float64), want)
    # products of 1 to 9 are whole multiples of 2^(2 - 13): the 8-bit instructions cut nothing off
    got = run_linear(hip_device, x, x_scales, w, w_scales, "float16")
    with np.errstate(over="ignore"):
        assert np.array_equal(got, want.astype(np.float32).astype(np.float16))


# Few steps of many columns: each of the kernels for one of the types at least, with rows and columns past its tiles' ends.
WIDE = [(13, 4099, 528), (27, 2051, 528), (27, 4099, 48), (61, 4099, 2064), (61, 4099, 528), (1, 24590, 144), (1, 24590, 528),
        (1, 24590, 2064), (77, 16390, 48), (77, 16390, 2064), (77, 16390, 528), (77, 8197, 4112), (150, 16390, 528),
        (205, 16390, 272), (205, 16390, 784), (602, 24590, 400), (1283, 6150, 48), (1283, 6150, 528)]


@pytest.mark.parametrize("out_dtype", ["float16", "float32"])
@pytest.mark.parametrize("shape", WIDE, ids=str)
def test_linear_of_many_columns(hip_device, shape, out_dtype):
    print(f"[case] linear {shape} {out_dtype}", flush=True)
    m, n, k = shape
    call = operands(sum(shape), *shape)
    got = run_linear(hip_device, *call, out_dtype)
    rows = np.unique(np.concatenate([np.arange(min(m, 5)), np.arange(max(m - 5, 0), m), np.random.default_rng(1).integers(0, m, 6)]))
    call, got = (call[0][rows], np.ascontiguousarray(call[1][:, rows]), *call[2:]), got[rows]
    plain.check_linear(got, *plain.linear(*call), k, plain.cut_off(*call) if out_dtype == "float16" else 0.0)


@pytest.mark.parametrize("shape", WIDE, ids=str)
def test_linear_of_whole_numbers_and_many_columns_is_exact(hip_device, shape):
    print(f"[case] linear {shape}", flush=True)
    test_linear_of_whole_numbers_is_exact(hip_device, shape)


@pytest.mark.parametrize("shape", [(1, 200, 400), (9, 200, 400), (40, 200, 400), (150, 300, 400), (600, 520, 400)], ids=str)
def test_linear_codes_that_are_not_numbers(hip_device, shape):
    """A NaN of x is in its row, one of w in its column, and nowhere else; so are scales that are not finite."""
    m, n, k = shape
    x, x_scales, w, w_scales = operands(5, m, n, k)
    x[m // 2, 399], w[n - 1, 130] = 0x7F, 0xFF
    w[3, 0] = 0x7F
    got = run_linear(hip_device, x, x_scales, w, w_scales, "float32")
    want, size = plain.linear(x, x_scales, w, w_scales)
    assert np.isnan(want).sum() == n + 2 * (m - 1)
    plain.check_linear(got, want, np.nan_to_num(size), k)
    x_scales[1, 0] = np.nan
    got = run_linear(hip_device, x, x_scales, w, w_scales, "float16")
    assert np.isnan(got[0]).all() and (m < 3 or not np.isnan(got[m - 1, 5:n - 1]).any())


def test_linear_results_repeat(hip_device):
    for shape in ((1, 4096, 4096), (24, 1000, 4096), (100, 640, 2048), (300, 500, 1024)):
        call = operands(1, *shape)
        first = run_linear(hip_device, *call, "float32")
        for _ in range(3):
            assert np.array_equal(run_linear(hip_device, *call, "float32"), first)
