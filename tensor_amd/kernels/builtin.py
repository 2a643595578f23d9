"""Manifests of the library's built-in executables by name."""

from __future__ import annotations

from tensor_amd.gguf import kernels as gguf
from tensor_amd.kernels import paged


def manifest(kernel: str, **options) -> dict:
    """The manifest of one built-in executable, GGUF or paged cache, with its options."""
    if kernel in paged.ENTRYPOINTS:
        return paged.manifest(kernel, **options)
    if kernel not in gguf.ENTRYPOINTS:
        raise ValueError(f"unknown HIP kernel {kernel!r}; choose {', '.join([*gguf.ENTRYPOINTS, *paged.ENTRYPOINTS])}")
    return gguf.manifest(kernel, **options)
