"""Operators that write a workspace, through torch on the GPU (tests/torch_scratch.py)."""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.timeout(300)
def test_workspaces_in_a_torch_first_process():
    print("[case] torch-scratch child", flush=True)
    result = subprocess.run([sys.executable, "-u", str(ROOT / "tests" / "torch_scratch.py")], cwd=ROOT,
                            capture_output=True, text=True, timeout=240, env=dict(os.environ, PYTHONPATH=str(ROOT)))
    print(result.stdout[-4000:], result.stderr[-4000:], flush=True)
    assert result.returncode == 0, result.stderr[-2000:]
    assert "[torch-scratch] ok" in result.stdout
