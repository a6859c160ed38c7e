"""The forms of the 16-bit experts' products stay within the tensor memory and the shared memory that they have (CPU:
the shapes' own constants, read by read)."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_reads_stay_within_what_is_there(tmp_path):
    exe = tmp_path / "product_shapes"
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "-I",
           str(ROOT / "libcusort_b200" / "csrc"), str(ROOT / "tests" / "cxx" / "product_shapes.cu"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout[-3000:] + r.stderr
