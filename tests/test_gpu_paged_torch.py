"""Paged-cache operators through the PyTorch binding, and the example that runs them together (tests/torch_paged.py)."""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.timeout(300)
@pytest.mark.parametrize("native", ["1", "0"], ids=["native-executor", "python-launch"])
def test_paged_operators_in_a_torch_first_process(native):
    print(f"[case] torch-paged child TENSOR_AMD_TORCH_NATIVE={native}", flush=True)
    result = subprocess.run([sys.executable, "-u", str(ROOT / "tests" / "torch_paged.py")], cwd=ROOT,
                            capture_output=True, text=True, timeout=240,
                            env=dict(os.environ, PYTHONPATH=str(ROOT), TENSOR_AMD_TORCH_NATIVE=native))
    print(result.stdout[-4000:], result.stderr[-4000:], flush=True)
    assert result.returncode == 0, result.stderr[-2000:]
    assert "[torch-paged] ok" in result.stdout
