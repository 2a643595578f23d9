"""Operators that write a workspace, checked by torch on the GPU and traced, run as its own process by
test_gpu_torch_scratch.py (torch is imported before the library)."""

from __future__ import annotations

import sys
from pathlib import Path

import torch  # first: the process's HIP runtime is torch's

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))

import tensor_amd.torch as tt  # noqa: E402
from tensor_amd.gguf.quant import sample_weight  # noqa: E402
from tensor_amd.torch.session import session  # noqa: E402
from tests.torch_paged import make, tensors  # noqa: E402


def step(name):
    print("[torch-scratch]", name, flush=True)


def group():
    """(kernel, inputs): two matrices on one input, enough rows that the sums go through the workspace."""
    m, k, rows = 96, 1024, (256, 128)
    x = torch.randn((m, k), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    weights = [torch.from_numpy(sample_weight(n, k, "q4_k", seed=i)).cuda() for i, n in enumerate(rows)]
    need = max(256, session(0).gemm_workspace("q4_k", m, k, rows))
    return tt.load("gguf_gemm_group", encoding="q4_k", count=2), [x, *weights, torch.zeros(need, dtype=torch.uint8, device="cuda")]


def attention():
    args = tensors(make(2, [1, 7, 40], [300, 90, 41], 33, 8, 2, 64, 16))
    args[-1].zero_()
    return tt.load("paged_attention"), args


def check(name, kernel, args):
    step(f"{name}: the operator's declaration")
    torch.library.opcheck(kernel._op, tuple(kernel._groups(args)), test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_static"))

    step(f"{name}: traced, the workspace read before and after")
    def call(*inputs):
        scratch = torch.zeros_like(inputs[-1])
        before = scratch.sum(dtype=torch.int64)
        out = kernel(*inputs[:-1], scratch)
        return before, scratch.sum(dtype=torch.int64), out

    torch.cuda.synchronize()
    want = call(*args)
    got = torch.compile(call, backend="aot_eager", fullgraph=True)(*args)
    assert int(got[0]) == 0 and int(got[1]) == int(want[1]), (got[:2], want[:2])
    for x, y in zip(*(v if isinstance(v, tuple) else (v,) for v in (got[2], want[2]))):
        assert torch.equal(x, y)
    return int(got[1])


if __name__ == "__main__":
    assert check("attention", *attention()) > 0
    check("group", *group())
    tt.close()
    print("[torch-scratch] ok", flush=True)
