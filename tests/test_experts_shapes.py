"""What the kernels of the experts' products read and write, worked out on the CPU by their own constants and
functions."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def _run(name, tmp_path):
    exe = tmp_path / name
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "-I",
           str(ROOT / "libcusort_b200" / "csrc"), str(ROOT / "tests" / "cxx" / f"{name}.cu"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout[-3000:] + r.stderr


def test_reads_stay_within_what_is_there(tmp_path):
    """Tensor memory and shared memory, by each form of the 16-bit products."""
    _run("product_shapes", tmp_path)


def test_rows_of_no_segment_are_those_that_are_cleared(tmp_path):
    _run("product_rows", tmp_path)
