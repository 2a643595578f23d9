"""Norm and 8-bit operators on torch tensors, run as its own process by test_gpu_fp8_torch.py.

torch is imported before the library is loaded, so both use one HIP runtime.  Each check prints its name before
it touches the GPU.
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch  # first: the process's HIP runtime is torch's

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))

import numpy as np  # noqa: E402

import tensor_amd.torch as tt  # noqa: E402
from examples import fp8_layer  # noqa: E402
from tensor_amd.kernels.fp8 import quantize_weight  # noqa: E402
from tests import fp8_cases as plain  # noqa: E402


def step(name):
    print("[torch-fp8]", name, flush=True)


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def host(x):
    return x.cpu().numpy()


def weights(seed, n, k):
    return quantize_weight(np.random.default_rng(seed).standard_normal((n, k)).astype(np.float32) * k ** -0.5)


def check_chain():
    """As a layer uses them: each operator's result on the one before it, against its own formula in 64 bits."""
    for tokens, hidden, inner in ((1, 512, 1024), (7, 384, 640), (150, 256, 400)):
        step(f"norm, linear, gates, linear: {tokens} tokens, {hidden} and {inner}")
        rng = np.random.default_rng(tokens)
        y = rng.standard_normal((tokens, hidden)).astype(np.float16)
        r = (3 * rng.standard_normal((tokens, hidden))).astype(np.float32)
        weight = rng.uniform(0.5, 1.5, hidden).astype(np.float32)
        codes, scales, stream = tt.load("rms_norm_fp8", residual="float32")(cuda(y), cuda(r), cuda(weight))
        want, h = plain.norm(y, r, weight, 1e-6)
        plain.check_codes(host(codes), host(scales), want, plain.NORM_OFF)
        plain.check_rounded(host(stream), h, "float32", 2.0 ** -24)
        # PyTorch's own type holds the same values
        assert np.array_equal(host(codes.view(torch.float8_e4m3fn).float()), plain.value(host(codes)).astype(np.float32))
        linear = tt.load("fp8_linear")
        w, ws = weights(1, 2 * inner, hidden)
        both = linear(codes, scales, cuda(w), cuda(ws))
        call = (host(codes), host(scales), w, ws)
        plain.check_linear(host(both), *plain.linear(*call), hidden, plain.cut_off(*call))
        codes, scales = tt.load("quantize_fp8", gated=True)(both)
        gates = host(both)
        plain.check_codes(host(codes), host(scales), plain.gated(gates), 2.0 ** -21 + 2.0 ** -23 * float(np.abs(gates).max()))
        w, ws = weights(2, hidden, inner)
        out = tt.load("fp8_linear", out_dtype="float32")(codes, scales, cuda(w), cuda(ws))
        call = (host(codes), host(scales), w, ws)
        plain.check_linear(host(out), *plain.linear(*call), inner)


def check_registered():
    step("registered operators, their fakes and what they refuse")
    linear = tt.load("fp8_linear")
    codes, scales = tt.load("quantize_fp8")(torch.randn((5, 272), device="cuda").half())
    w, ws = (cuda(t) for t in weights(3, 300, 272))
    out = linear(codes, scales, w, ws)
    again = torch.empty_like(out)
    linear.into(codes, scales, w, ws, outputs=[again])
    assert torch.equal(out, again)
    (fake,) = linear.fake([codes, scales, w, ws])
    assert fake.shape == out.shape and fake.dtype == out.dtype
    for wrong in ((codes[:, :256].contiguous(), scales, w, ws), (codes, scales.t().contiguous(), w, ws),
                  (codes, scales, w[:, :264].contiguous(), ws), (codes, scales, w, ws[:1].contiguous()),
                  (codes.view(torch.float8_e4m3fn), scales, w, ws), (codes.t(), scales, w, ws)):
        try:
            linear.raw(*wrong)
        except (ValueError, TypeError):
            continue
        raise AssertionError("a call of the wrong shapes or types ran")


def check_surroundings():
    step("memory around the outputs stays as it is")
    for m, n, k in ((1, 40, 128), (3, 1000, 272), (40, 129, 400), (77, 250, 2544), (200, 300, 272), (600, 1300, 144)):
        codes, scales = tt.load("quantize_fp8")(torch.randn((m, k), device="cuda").half())
        w, ws = (cuda(t) for t in weights(4, n, k))
        for dtype in (torch.float16, torch.float32):
            room = torch.full((m * n + 2048,), 7.0, dtype=dtype, device="cuda")
            out = room[1024:1024 + m * n].view(m, n)
            linear = tt.load("fp8_linear", out_dtype=str(dtype).removeprefix("torch."))
            linear.prepare(codes, scales, w, ws, outputs=[out])()
            assert torch.equal(out, linear(codes, scales, w, ws))
            assert bool((room[:1024] == 7.0).all()) and bool((room[1024 + m * n:] == 7.0).all()), (m, n, k)
    for rows, width in ((3, 100), (5, 128), (2, 1000), (3, 4100), (1, 9001)):
        x = torch.randn((rows, width), device="cuda").half()
        room = torch.full((rows * width + 2048,), 7, dtype=torch.uint8, device="cuda")
        codes, scales = room[1024:1024 + rows * width].view(rows, width), torch.empty((-(-width // 128), rows), device="cuda")
        for kernel, args in ((tt.load("quantize_fp8"), (x,)), (tt.load("rms_norm_fp8"), (x, torch.ones(width, device="cuda")))):
            room.fill_(7)
            kernel.prepare(*args, outputs=[codes, scales])()
            want = kernel(*args)
            assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
            assert bool((room[:1024] == 7).all()) and bool((room[1024 + rows * width:] == 7).all()), (rows, width)


def check_streams():
    step("a stream of its own")
    linear, quantize = tt.load("fp8_linear"), tt.load("quantize_fp8")
    x, (w, ws) = torch.randn((100, 2048), device="cuda").half(), (cuda(t) for t in weights(5, 1000, 2048))
    want = linear(*quantize(x), w, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [t.clone() for t in (x, w, ws)]  # made on the side stream, in its order
        out = linear(*quantize(late[0]), *late[1:])
        del late
        junk = torch.full((1 << 20,), 7.0, device="cuda")  # what those tensors' memory may hold next
    side.synchronize()
    assert torch.equal(out, want) and bool((junk == 7.0).all())


def check_graph():
    step("a captured step, replayed")
    norm, linear, gated = tt.load("rms_norm_fp8", residual="float16"), tt.load("fp8_linear"), tt.load("quantize_fp8", gated=True)
    for tokens in (1, 12, 90):
        y, r = (torch.randn((tokens, 512), device="cuda").half() for _ in range(2))
        weight = torch.rand(512, device="cuda") + 0.5
        up, down = ([cuda(t) for t in weights(seed, n, k)] for seed, n, k in ((6, 1280, 512), (7, 512, 640)))
        first = norm.prepare(y, r, weight)
        second = linear.prepare(*first.outputs[:2], *up)
        third = gated.prepare(second.outputs[0])
        last = linear.prepare(*third.outputs, *down)
        calls = (first, second, third, last)
        for call in calls:
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for call in calls:
                call()
        for replay in range(3):
            last.outputs[0].zero_()
            y.mul_(-1.5 if replay else 1.0)
            codes, scales, _ = norm(y, r, weight)
            want = linear(*gated(linear(codes, scales, *up)), *down)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(last.outputs[0], want), (tokens, replay)


def whole(n, k):
    """Codes of 0, 1, 2 and their negatives: sums of up to 2^20 products are whole numbers below 2^22, exact in any order."""
    codes = torch.tensor([0x00, 0x38, 0x40, 0xB8, 0xC0], dtype=torch.uint8, device="cuda")
    return codes[torch.randint(0, 5, (n, k), device="cuda")]


def ones(*shape):
    return torch.ones(shape, device="cuda")


def check_far():
    """Places past 2^32 and the longest extents."""
    for m, n, k, dtype in ((140001, 32770, 16, "float16"), (70001, 32770, 48, "float32"), (1 << 20, 40, 16, "float16"),
                           (1, 1 << 22, 16, "float32"), (70, 1 << 22, 32, "float16")):
        step(f"linear {m} x {n} x {k} {dtype}")
        linear, x, w = tt.load("fp8_linear", out_dtype=dtype), whole(m, k), whole(n, k)
        ws = ones(-(-n // 128), 1)
        out = linear(x, ones(1, m), w, ws)
        rows = torch.unique(torch.cat([torch.arange(min(m, 9)), torch.arange(max(m - 9, 0), m), torch.randint(0, m, (20,))])).cuda()
        want = linear(x[rows], ones(1, len(rows)), w, ws)
        assert torch.equal(out[rows], want)
        columns = torch.unique(torch.cat([torch.arange(min(n, 9)), torch.arange(n - 9, n), torch.randint(0, n, (20,))])).cuda()
        values = torch.from_numpy(plain.value(np.arange(256))).cuda()
        exact = values[x[rows].long()] @ values[w[columns].long()].T
        assert torch.equal(out[rows][:, columns].double(), exact)
        del out, want
    for dtype in ("float16", "float32"):
        step(f"linear 3 x 130 x {1 << 20} {dtype}")
        k = 1 << 20
        x, w = whole(3, k), whole(130, k)
        out = tt.load("fp8_linear", out_dtype=dtype)(x, ones(k // 128, 3), w, ones(2, k // 128))
        values = torch.from_numpy(plain.value(np.arange(256))).cuda()
        exact = values[x.long()] @ values[w.long()].T
        assert torch.equal(out, exact.to(out.dtype))
    step("gates of 110001 x 24576")
    x = torch.randn((110001, 2 * 24576), device="cuda", dtype=torch.float16)
    codes, scales = tt.load("quantize_fp8", gated=True)(x)
    want, want_scales = tt.load("quantize_fp8", gated=True)(x[-100:])
    assert torch.equal(codes[-100:], want) and torch.equal(scales[:, -100:], want_scales)
    del codes, scales, want
    step("norm of 220002 x 24576")
    x = x.view(220002, 24576)
    weight = torch.rand(24576, device="cuda")
    out = tt.load("rms_norm")(x, weight)
    assert torch.equal(out[-100:], tt.load("rms_norm")(x[-100:], weight))
    del x, out
    torch.cuda.empty_cache()


def check_surroundings_of_tiles():
    step("memory around the outputs of each kind of tile")
    for m, n, k in ((1, 24590, 528), (1, 24590, 2064), (77, 16390, 528), (77, 8197, 4112), (150, 16390, 528), (205, 16390, 784),
                    (1283, 6150, 528)):
        x, w, xs, ws = whole(m, k), whole(n, k), ones(-(-k // 128), m), ones(-(-n // 128), -(-k // 128))
        for dtype in ("float16", "float32"):
            room = torch.full((m * n + 131072,), 7.0, dtype=getattr(torch, dtype), device="cuda")
            out = room[65536:65536 + m * n].view(m, n)
            linear = tt.load("fp8_linear", out_dtype=dtype)
            linear.prepare(x, xs, w, ws, outputs=[out])()
            assert torch.equal(out, linear(x, xs, w, ws))
            assert bool((room[:65536] == 7.0).all()) and bool((room[65536 + m * n:] == 7.0).all()), (m, n, k)


def check_example():
    # the weights are the codes' own; activations are rounded to 8 bits four times on the way (2^-4 at most, evenly spread
    # errors of 2^-4 / sqrt(3) in the 2-norm and less), and what they add to stays
    for options in (dict(requests=4, steps=4), dict(requests=9, steps=2, hidden=640, inner=1200, heads=4, kv=4, page=8)):
        step(f"layer of the example {options}")
        assert fp8_layer.run(**options) < 4 * 2.0 ** -4


if __name__ == "__main__":
    check_chain()
    check_registered()
    check_surroundings()
    check_streams()
    check_graph()
    check_far()
    check_surroundings_of_tiles()
    check_example()
    tt.close()
    print("[torch-fp8] ok", flush=True)
