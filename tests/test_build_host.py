"""When the library and its PyTorch binding are built anew (no compiler and no GPU needed)."""
from __future__ import annotations

import os
import time

import pytest

from libcusort_b200 import build as b


@pytest.fixture
def built(tmp_path, monkeypatch):
    """A finished build in a folder of its own, newer than every source, beside a PyTorch with CUDA."""
    torch = tmp_path / "torch"
    (torch / "lib").mkdir(parents=True)
    (torch / "lib" / "libc10_cuda.so").touch()
    for name, path in (("LIB", tmp_path / "lib.so"), ("BINDING", tmp_path / "binding.so"),
                       ("STAMP", tmp_path / "stamp.txt")):
        monkeypatch.setattr(b, name, path)
        path.touch()
    monkeypatch.setattr(b, "torch_dir", lambda: torch)
    b.STAMP.write_text(b.stamp())
    now = time.time() + 100
    os.utime(b.LIB, (now, now))
    os.utime(b.BINDING, (now + 5, now + 5))
    assert b.up_to_date()
    return torch


def test_binding_older_than_the_library(built):
    """As a failed compilation of the binding leaves it."""
    before = b.LIB.stat().st_mtime - 1
    os.utime(b.BINDING, (before, before))
    assert not b.up_to_date()


def test_binding_missing(built):
    b.BINDING.unlink()
    assert not b.up_to_date()


def test_other_pytorch(built, monkeypatch):
    monkeypatch.setattr(b, "torch_version", lambda: "0.0.1")
    assert not b.up_to_date()


def test_other_defines(built, monkeypatch):
    monkeypatch.setenv("CUSORT_NVCC_DEFINES", "-DCUSORT_TEST_ONLY=1")
    assert not b.up_to_date()


@pytest.mark.parametrize("there", [True, False])
def test_pytorch_without_cuda(built, monkeypatch, capsys, there):
    """The library is built alone where no PyTorch, or one without CUDA, is installed."""
    (built / "lib" / "libc10_cuda.so").unlink()
    if not there:
        monkeypatch.setattr(b, "torch_dir", lambda: None)
    b.BINDING.unlink()
    b._build_binding()
    assert not b.BINDING.exists() and "is not built" in capsys.readouterr().err
    b.STAMP.write_text(b.stamp())
    assert b.up_to_date()
