"""Build the CUDA library in-tree: libcusort_b200/_lib/libcusort_b200.so.

Every .cu under csrc/ is compiled for sm_100a only
(-gencode arch=compute_100a,code=sm_100a) in parallel, then linked into one
shared library with the CUDA runtime linked statically and NCCL dynamically.
Where a PyTorch with CUDA is installed, csrc/torch_binding.cpp is compiled beside it
(libcusort_b200/_lib/_cusort_torch.so): the native half of the routing and
placement operators' Python functions, over the same C ABI.
Run as ``python -m libcusort_b200.build`` or through ``__graft_entry__.build()``.

Environment CUSORT_NVCC_DEFINES adds preprocessor definitions to every
compile (e.g. ``-DCUSORT_LOOKBACK_TIMER=1`` for the lookback-timer build that
``bench.py --lookback-stall`` reads); the definitions of the last build
and the version of PyTorch are kept beside the library, so a change of them
forces a rebuild.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT_DIR = PKG / "_lib"
OBJ_DIR = PKG / "_build"
LIB = OUT_DIR / "libcusort_b200.so"
BINDING = OUT_DIR / "_cusort_torch.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
              "--expt-relaxed-constexpr"]
STAMP = OUT_DIR / "defines.txt"


def extra_defines() -> list[str]:
    """-D flags from CUSORT_NVCC_DEFINES (anything else there is rejected)."""
    flags = os.environ.get("CUSORT_NVCC_DEFINES", "").split()
    bad = [f for f in flags if not f.startswith("-D")]
    if bad:
        raise ValueError(f"CUSORT_NVCC_DEFINES takes -D flags only, got {bad}")
    return flags


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def nccl_flags() -> list[str]:
    """Header + library location of NCCL (system install)."""
    inc = []
    for d in ("/usr/include", "/usr/local/cuda/include"):
        if Path(d, "nccl.h").exists():
            inc = ["-I" + d]
            break
    return inc


def _compile(src: Path, verbose: bool) -> tuple[Path, str]:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, *extra_defines(), *nccl_flags(), "-Xptxas", "-v", "-c", str(src), "-o",
           str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stderr}")
    return obj, r.stderr


def torch_dir() -> Path | None:
    """Where PyTorch's headers and libraries lie (found without importing it)."""
    spec = importlib.util.find_spec("torch")
    return Path(list(spec.submodule_search_locations)[0]) if spec else None


def torch_version() -> str:
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return ""


def binding_possible() -> bool:
    """Whether a PyTorch with CUDA is there to build the binding against."""
    t = torch_dir()
    return t is not None and (t / "lib" / "libc10_cuda.so").exists()


def _build_binding() -> None:
    if not binding_possible():
        print("no PyTorch with CUDA is installed: the PyTorch binding is not built", file=sys.stderr)
        return
    t = torch_dir()
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-sign-compare",
           "-I" + sysconfig.get_paths()["include"], "-isystem", str(t / "include"), "-isystem",
           str(t / "include" / "torch" / "csrc" / "api" / "include"), "-isystem", str(cuda / "include"),
           str(CSRC / "torch_binding.cpp"), "-o", str(tmp), "-L" + str(t / "lib"), "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-L" + str(OUT_DIR), "-l:" + LIB.name,
           "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for torch_binding.cpp:\n{r.stderr}")
    os.replace(tmp, BINDING)


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def stamp() -> str:
    """What else than the sources a build depends on."""
    return "\n".join([" ".join(extra_defines()), "torch " + torch_version() if binding_possible() else "no binding"])


def up_to_date() -> bool:
    if not LIB.exists() or (STAMP.read_text() if STAMP.exists() else "") != stamp():
        return False
    t = LIB.stat().st_mtime
    # the binding is compiled after the library is linked: an older one is left over from before a failure
    if binding_possible() and not (BINDING.exists() and BINDING.stat().st_mtime >= t):
        return False
    deps = list(CSRC.glob("*")) + [PKG.parent / "include" / "cusort_b200.h", Path(__file__)]
    return all(p.stat().st_mtime <= t for p in deps if p.exists())


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return LIB
    OUT_DIR.mkdir(exist_ok=True)
    OBJ_DIR.mkdir(exist_ok=True)
    srcs = sources()
    logs = []
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = []
        for obj, log in ex.map(lambda s: _compile(s, verbose), srcs):
            objs.append(obj)
            logs.append(log)
    (OBJ_DIR / "ptxas.log").write_text("".join(logs))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lnccl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    _build_binding()
    STAMP.write_text(stamp())
    if verbose:
        print("".join(logs))
    return LIB


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(p)
