"""Manifests of the library's built-in executables by name."""

from __future__ import annotations

from tensor_amd.gguf import kernels as gguf
from tensor_amd.kernels import fp8, paged


def manifest(kernel: str, **options) -> dict:
    """The manifest of one built-in executable, GGUF, paged cache, norm or 8-bit, with its options."""
    for module in (paged, fp8):
        if kernel in module.ENTRYPOINTS:
            return module.manifest(kernel, **options)
    if kernel not in gguf.ENTRYPOINTS:
        names = [*gguf.ENTRYPOINTS, *paged.ENTRYPOINTS, *fp8.ENTRYPOINTS]
        raise ValueError(f"unknown HIP kernel {kernel!r}; choose {', '.join(names)}")
    return gguf.manifest(kernel, **options)
