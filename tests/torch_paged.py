"""Paged-cache operators on torch tensors, run as its own process by test_gpu_paged_torch.py.

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
from examples import paged_decode  # noqa: E402
from tensor_amd.kernels.paged import rotary_angles  # noqa: E402
from tensor_amd.torch.session import session  # noqa: E402
from tests import paged_cases as plain  # noqa: E402


def step(name):
    print("[torch-paged]", name, flush=True)


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def make(seed, counts, lengths, prefix, heads, kv, dim, page):
    rng = np.random.default_rng(seed)
    table, prefix_pages, pages = plain.paging(rng, lengths, page, prefix)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rng.standard_normal((offsets[-1], heads, dim)).astype(np.float16)
    caches = rng.standard_normal((2, pages, kv, page, dim)).astype(np.float16)
    return [q, caches[0], caches[1], offsets, np.asarray(lengths, np.int32), table, prefix_pages, prefix]


def tensors(call):
    """The operator's inputs: the arrays on the GPU, the prefix's length as one, a workspace."""
    q, k = call[0], call[1]
    need = session(0).attention_workspace(q.shape[0], len(call[4]), q.shape[1], k.shape[1], q.shape[2])
    return [cuda(x) for x in call[:7]] + [cuda(np.array([call[7]], np.int32)), torch.empty(need, dtype=torch.uint8, device="cuda")]


def check_example():
    for options in (dict(requests=4, steps=4, prefix=50), dict(requests=9, steps=2, prefix=16, heads=4, kv=4, dim=64, page=8)):
        step(f"layer of the example {options}")
        assert paged_decode.run(**options) <= 1.0


def check_operators():
    step("registered operators")
    call = make(1, [1, 7, 40], [30, 90, 41], 33, 8, 2, 64, 16)
    want, bound = plain.attention(*call)
    attention = tt.load("paged_attention")
    args = tensors(call)
    out = attention(*args)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
    again = torch.empty_like(out)
    attention.into(*args, outputs=[again])
    assert torch.equal(out, again)
    (fake,) = attention.fake(args)
    assert fake.shape == out.shape and fake.dtype == out.dtype

    step("rotary there and back")
    angles = cuda(rotary_angles(64, 64))
    q, k = args[0], args[1][:, 0, 0, :].reshape(-1, 1, 64).repeat(q_rows(args[0], args[1]), 1, 1)[:args[0].shape[0]].contiguous()
    at = torch.arange(q.shape[0], dtype=torch.int32, device="cuda")
    turned = tt.load("rotary")(q, k, at, angles)
    back = tt.load("rotary", inverse=True)(*turned, at, angles)
    # two rotations, each rounded to fp16: 2^-11 of a pair's length each, and fp32's own
    for x, y in zip((q, k), back):
        pair = torch.hypot(x[..., :32].double(), x[..., 32:].double()).repeat(1, 1, 2)
        assert bool(((x.double() - y.double()).abs() <= 2.0 ** -9 * pair + 2.0 ** -23).all())


def q_rows(q, cache):
    return -(-q.shape[0] // cache.shape[0])


def check_store_is_not_functional():
    step("rotary_store updates its inputs")
    store = tt.load("rotary_store")
    tokens, heads, kv, dim, pages, page = 5, 4, 2, 64, 3, 8
    g = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn((tokens, n, dim), device="cuda", generator=g).half() for n in (heads, kv, kv))
    caches = [torch.zeros((pages, kv, page, dim), dtype=torch.float16, device="cuda") for _ in range(2)]
    at, slots = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1, 2, 3, 4], [9, 23, -1, 0, 1]))
    args = (q, k, v, at, slots, cuda(rotary_angles(8, dim)), torch.empty_like(q), *caches)
    try:
        store(*args)
    except Exception as error:  # noqa: BLE001
        assert type(error).__name__ in ("RuntimeError", "TypeError", "ValueError"), error
    else:
        raise AssertionError("rotary_store ran as a functional operator")
    assert not any(bool(c.any()) for c in caches)
    store.raw(*args)
    for t, slot in enumerate((9, 23, -1, 0, 1)):
        if slot >= 0:
            assert torch.equal(caches[1][slot // page, :, slot % page], v[t])
    assert int((caches[1].abs().sum(-1) > 0).sum()) == 4 * kv


def check_streams():
    step("a stream of its own")
    attention = tt.load("paged_attention")
    call = make(5, [1] * 6, [100, 3, 77, 200, 31, 64], 65, 8, 2, 128, 16)
    want, bound = plain.attention(*call)
    args = tensors(call)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [x.clone() for x in args]  # made on the side stream, in its order
        out = attention(*late)
        del late
        junk = torch.full((1 << 20,), 7.0, device="cuda")  # what those tensors' memory may hold next
    side.synchronize()
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all() and bool((junk == 7.0).all())


def check_graph():
    step("a captured step, replayed")
    attention = tt.load("paged_attention")
    call = make(6, [1] * 4 + [33], [100, 3, 77, 200, 64], 65, 8, 2, 128, 16)
    args = tensors(call)
    prepared = attention.prepare(*args)
    eager = attention(*args)
    prepared()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prepared()
    out = prepared.outputs[0]
    for replay in range(3):
        out.zero_()
        args[0].mul_(-1.0 if replay else 1.0)
        want = attention(*args[:8], args[8].clone())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), replay
        if replay == 0:
            assert torch.equal(out, eager)


if __name__ == "__main__":
    check_operators()
    check_store_is_not_functional()
    check_streams()
    check_graph()
    check_example()
    tt.close()
    print("[torch-paged] ok", flush=True)
