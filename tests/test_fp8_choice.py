"""Which kernel an 8-bit linear takes (csrc/fp8_choice.h), compiled as plain host code (CPU only): the calls that test each tile
kernel on a GPU take it, and cover what can go wrong in it."""

from __future__ import annotations

import ctypes as c
import subprocess
from pathlib import Path

import pytest

from tests import fp8_tiles
from tests.test_gpu_fp8 import SHAPES, WIDE

CSRC = Path(__file__).resolve().parents[1] / "tensor_amd" / "csrc"
SOURCE = """
#include "fp8_choice.h"
using namespace tensor_fp8;
extern "C" int kernel(int m, int n, int k, int f32) { return linear_kernel(m, n, k, f32); }
extern "C" int tile(int kernel, int f32, int* out) {
  const int count = f32 ? sizeof(kLinearFp32) / sizeof(LinearCost) : sizeof(kLinearFp16) / sizeof(LinearCost);
  if (kernel >= count) return 0;
  const LinearCost& cost = f32 ? kLinearFp32[kernel] : kLinearFp16[kernel];
  out[0] = cost.bn, out[1] = cost.bm;
  return 1;
}
"""


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    folder = tmp_path_factory.mktemp("fp8_choice")
    (folder / "choice.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(CSRC),
                    str(folder / "choice.cpp"), "-o", str(folder / "choice.so")], check=True, capture_output=True)
    return c.CDLL(str(folder / "choice.so"))


def test_kernels_are_those_of_the_library(library):
    for dtype, kernels in fp8_tiles.KERNELS.items():
        f32, out = int(dtype == "float32"), (c.c_int * 2)()
        assert not library.tile(max(kernels) + 1, f32, out)
        for kernel, (bn, bm, _, _) in kernels.items():
            assert library.tile(kernel, f32, out) and tuple(out) == (bn, bm)


@pytest.mark.parametrize("case", fp8_tiles.CASES, ids=str)
def test_calls_take_the_kernel_that_they_test(library, case):
    dtype, kernel, shape = case
    assert library.kernel(*shape, int(dtype == "float32")) == kernel


def test_every_tile_kernel_is_covered(library):
    for dtype, kernels in fp8_tiles.KERNELS.items():
        for kernel, (bn, bm, stages, alone) in kernels.items():
            shapes = [shape for d, i, shape in fp8_tiles.CASES if (d, i) == (dtype, kernel)]
            for short in (False, True):
                mine = [(m, n, -(-k // 128)) for m, n, k in shapes if bool(k % 128) == short]
                # the main loop, from its second tiles on, with rows past the ends of the last ones
                assert any(steps >= fp8_tiles.main_steps(stages, alone) and m > bm and m % bm and n > bn and n % bn
                           for m, n, steps in mine), (dtype, kernel, short)
        assert {i for d, i, _ in fp8_tiles.LONG if d == dtype} == set(kernels)


def test_kernels_of_few_rows_are_taken(library):
    """Each of them by some call of the other tests."""
    for f32 in (0, 1):
        taken = {library.kernel(*shape, f32) for shape in SHAPES + WIDE}
        assert set(range(5)) <= taken, taken


def test_the_largest_extents_have_a_kernel_whose_launch_they_fit(library):
    """At most 2^22 workgroups of any of the kernels, and the extents that the entry point takes."""
    for m, n in ((1 << 20, 1 << 15), (1 << 13, 1 << 22), (1, 1 << 22), (1 << 20, 1), (1 << 17, 1 << 18), ((1 << 20) - 1, (1 << 15) - 1)):
        for k in (16, 1 << 20):
            for f32 in (0, 1):
                out = (c.c_int * 2)()
                assert library.tile(library.kernel(m, n, k, f32), f32, out)
                assert -(-n // out[0]) * -(-m // out[1]) <= 1 << 22, (m, n, k, f32)
