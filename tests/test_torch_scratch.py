"""Kernels that write a workspace among their inputs: their registered operators say so (CPU only, fake tensors)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

import tensor_amd.torch as tt  # noqa: E402
from tensor_amd.gguf.kernels import manifest  # noqa: E402
from tests.test_torch_bridge import fake, row_bytes  # noqa: E402


def attention_inputs():
    ints = [fake(*shape, dtype=torch.int32) for shape in ((3,), (2,), (2, 4), (1,), (1,))]
    return [fake(3, 8, 64), fake(5, 2, 16, 64), fake(5, 2, 16, 64), *ints, fake(1 << 20, dtype=torch.uint8)]


def group_inputs(count):
    return [fake(16, 512), *(fake(8 * (i + 1), row_bytes("q4_k", 512), dtype=torch.uint8) for i in range(count)),
            fake(4096, dtype=torch.uint8)]


CASES = {"attention": ("paged_attention", {}, attention_inputs, [(3, 8, 64)]),
         "group of 1": ("gguf_gemm_group", dict(encoding="q4_k", count=1), lambda: group_inputs(1), [(16, 8)]),
         "group of 3": ("gguf_gemm_group", dict(encoding="q4_k", count=3), lambda: group_inputs(3), [(16, 8), (16, 16), (16, 24)])}


@pytest.mark.parametrize("case", CASES)
def test_a_workspace_counts_as_written(case):
    name, options, inputs, shapes = CASES[case]
    kernel = tt.load(name, **options)
    with FakeTensorMode():
        args = inputs()
        before = [a._version for a in args]
        outs = kernel(*args)
        outs = [outs] if len(shapes) == 1 else outs
        assert [tuple(o.shape) for o in outs] == shapes
        assert [a._version - b for a, b in zip(args, before)] == [0] * (len(args) - 1) + [1]
        kernel.into(*args, outputs=[fake(*shape) for shape in shapes])
        assert [a._version - b for a, b in zip(args, before)] == [0] * (len(args) - 1) + [2]


def test_scratch_names_input_buffers():
    for name in ("out", "type", "nothing"):
        with pytest.raises(ValueError, match="scratch"):
            tt.Kernel(dict(manifest("gguf_linear", "q4_k"), scratch=[name]))
