"""The sources with inline assembly compile for gfx950 without a warning: the code generator
warns where a statement's operands or clobbers are not what the compiler can honour."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "neurosim-gpu_amd" / "csrc"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc is not installed")
@pytest.mark.parametrize("source", ["mx_product.hip", "scan.hip", "scan_grad.hip"])
def test_kernels_compile_without_warnings(tmp_path, source):
    build = [HIPCC, "-O1", "-std=c++17", "--offload-arch=gfx950", "--offload-device-only", "-S",
             f"-I{ROOT / 'include'}", f"-I{CSRC}", "-Xclang", "-target-feature", "-Xclang",
             "-packed-fp32-ops", "-Wall", "-Wno-unused-function", "-Wno-unused-command-line-argument",
             str(CSRC / source), "-o", str(tmp_path / "kernels.s")]
    run = subprocess.run(build, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-4000:]
    assert "warning:" not in run.stderr, run.stderr[-4000:]
