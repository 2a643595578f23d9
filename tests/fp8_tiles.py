"""Calls of the 8-bit linear that take each of its tile kernels: whole steps of K and a short last one, fewer steps than the kernel
has stages and as many as its main loop needs, several tiles in both directions with rows past the last ones' ends.

``test_fp8_choice.py`` holds the kernels to them, ``test_gpu_fp8_tiles.py`` runs them.
"""

from __future__ import annotations

# of a kernel: weight rows and activation rows of a tile, stages, whether its multiplying waves load for themselves
KERNELS = {
    "float16": {5: (64, 64, 4, False), 6: (128, 64, 3, False), 7: (128, 128, 4, False), 8: (256, 128, 3, False),
                9: (256, 256, 2, True)},
    "float32": {5: (64, 64, 4, False), 6: (64, 64, 4, True), 7: (128, 64, 3, False), 8: (128, 64, 3, True),
                9: (128, 128, 4, False), 10: (128, 128, 2, True)},
}


def main_steps(stages, alone):
    """Steps of K from which on a kernel goes through its main loop."""
    return 2 * stages + 1 if alone else stages


# kernel: (m, n), steps of fewer than its stages that it is taken for, steps of its main loop and some after it
_SIZES = {
    "float16": {5: ((547, 451), (1, 2, 3), (5, 7)), 6: ((69, 16427), (1, 2), (4, 6)), 7: ((133, 11051), (), (15, 18)),
                8: ((195, 16427), (), (7, 8)), 9: ((387, 18731), (1, 2), (6, 9))},
    "float32": {5: ((69, 4139), (1, 2, 3), (5, 7)), 6: ((69, 8235), (), (10, 12)), 7: ((69, 8235), (), (29, 30)),
                8: ((133, 16427), (1, 2), (8, 9)), 9: ((133, 11051), (1, 2, 3), (5, 7)), 10: ((195, 16427), (1, 2), (6, 9))},
}

# (type of the results, kernel, (m, n, k))
CASES = [(dtype, kernel, (*size, 128 * steps - short))
         for dtype, kernels in _SIZES.items() for kernel, (size, few, many) in kernels.items()
         for steps in (*few, *many) for short in (0, 48)]
CASES.append(("float16", 7, (333, 6144, 4096)))

# those of a main loop, one of whole steps and one of a short last step for each kernel
LONG = [(dtype, kernel, (*size, 128 * steps - short)) for dtype, kernels in _SIZES.items()
        for kernel, (size, _, many) in kernels.items() for steps, short in zip(many, (0, 48))]
