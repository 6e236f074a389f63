"""Build step for the sm_100a C-ABI library ``_lib/libnimbleml_tied_ce.so``.

The library is compiled in-tree with nvcc for ``sm_100a`` only (tcgen05 /
TMA code has no portable fallback), linked against the static CUDA runtime,
and resolves the driver's ``cuTensorMapEncodeTiled`` at run time, so the .so
loads on hosts without a GPU. Run ``python -m nimbleml_b200.build_native``.

The same step builds ``_lib/nimbleml_tied_ce_native*.so``, the pybind11
module with the reference-style ``*_device`` entry points
(``csrc/tied_ce_pybind.cpp``), linked against the library with an
``$ORIGIN`` run path, and ``_lib/nimbleml_b200_host.torch-<version>*.so``, the
torch host side of the operators whose calls are short (``csrc/torch_host.cpp``),
one file for each torch version.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libnimbleml_tied_ce.so"
SOURCES = [CSRC / "tied_ce.cu", CSRC / "rowwise.cu", CSRC / "token_logprobs.cu", CSRC / "layernorm.cu",
           CSRC / "adamw_many.cu"]
HEADERS = [CSRC / "sm100_ptx.cuh", CSRC / "common.cuh", CSRC / "elementwise.cuh",
           REPO_DIR / "include" / "nimbleml_tied_ce.h"]
PYBIND_SOURCE = CSRC / "tied_ce_pybind.cpp"
HOST_SOURCE = CSRC / "torch_host.cpp"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-cudart", "static", "--threads", "0",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")


def pybind_module_path() -> Path:
    ext = sysconfig.get_config_var("EXT_SUFFIX") or ".so"
    return LIB_DIR / f"nimbleml_tied_ce_native{ext}"


def host_module_path() -> Path:
    """The host module of the installed torch: it is compiled against torch's headers, so one that was built
    with another version is not this one (it is neither loaded nor taken for up to date)."""
    import torch

    ext = sysconfig.get_config_var("EXT_SUFFIX") or ".so"
    return LIB_DIR / f"nimbleml_b200_host.torch-{torch.__version__}{ext}"


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    built = target.stat().st_mtime
    return any(p.stat().st_mtime > built for p in deps)


def build_pybind(force: bool = False, verbose: bool = False) -> Path:
    """Compile the pybind11 module (g++) if it is older than its source or the library."""
    out = pybind_module_path()
    if not force and not _stale(out, [PYBIND_SOURCE, LIB_PATH, HEADERS[-1]]):
        return out
    import pybind11

    tmp = out.with_suffix(".tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           "-I", pybind11.get_include(), "-I", sysconfig.get_paths()["include"], "-I", str(REPO_DIR / "include"),
           str(PYBIND_SOURCE), "-L", str(LIB_DIR), "-l:" + LIB_PATH.name, "-Wl,-rpath,$ORIGIN", "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, out)
    return out


def build_host(force: bool = False, verbose: bool = False) -> Path:
    """Compile the torch host module (g++ against the installed torch) if there is none for this torch, or one older
    than its source or the library."""
    out = host_module_path()
    if not force and not _stale(out, [HOST_SOURCE, LIB_PATH, HEADERS[-1]]):
        return out
    import torch

    base = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parents[1]
    tmp = out.with_suffix(".tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-I", str(base / "include"), "-I", str(base / "include" / "torch" / "csrc" / "api" / "include"),
           "-I", str(cuda / "include"), "-I", sysconfig.get_paths()["include"], "-I", str(REPO_DIR / "include"),
           str(HOST_SOURCE), "-L", str(LIB_DIR), "-l:" + LIB_PATH.name, "-L", str(base / "lib"), "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch", "-ltorch_python",
           # The shared C++ runtime that torch uses, by its file name: a compiler whose libstdc++.so link is missing
           # would take the static one, and two copies of its locale facets break the first formatted message.
           "-l:libstdc++.so.6", "-Wl,-rpath,$ORIGIN", "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, out)
    return out


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if a source is newer than the .so (or ``force``), then the two host modules."""
    if force or _stale(LIB_PATH, SOURCES + HEADERS):
        LIB_DIR.mkdir(parents=True, exist_ok=True)
        tmp = LIB_PATH.with_suffix(".so.tmp")
        cmd = [_nvcc(), *NVCC_FLAGS, "-I", str(REPO_DIR / "include"), "-o", str(tmp), *map(str, SOURCES)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB_PATH)
    build_pybind(force=force, verbose=verbose)
    build_host(force=force, verbose=verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
