"""Build ``libq3b200.so`` (every CUDA/C++ source under ``csrc/``) for sm_100a, and
``_native.so``, the Python side of its rotary and paged-chunk operators
(``csrc/python/``, against the torch that this interpreter imports).

    python qwen3-tile-ops_b200/build.py          # incremental
    python qwen3-tile-ops_b200/build.py --clean

nvcc cross-compiles without a GPU.  Objects go to ``_build/`` and the shared
library lands next to this file, where the Python package loads it from.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libq3b200.so"
NATIVE = PKG / "_native.so"
INCLUDE = PKG.parent / "include"

NVCC = os.environ.get("NVCC", "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-fmad=false", "-Xcompiler", "-fPIC",
         "-Xptxas", "-warn-spills", f"-I{INCLUDE}", f"-I{CSRC}"]


def _deps(src: Path) -> list[Path]:
    return sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.inc")) + \
        [INCLUDE / "q3_ops.h", src]


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    if obj.exists() and all(obj.stat().st_mtime >= d.stat().st_mtime for d in _deps(src)):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    if verbose or "spill" in res.stderr.lower():
        sys.stderr.write(res.stderr)
    return obj


def _native(lib: Path) -> None:
    """``_native.so`` next to the library, which it finds by its own place.  A host that uses the
    C ABI alone may lack what it is built against: then the library is all there is."""
    import sysconfig

    missing = None
    try:
        import torch
    except ImportError as e:
        missing = str(e)
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        missing = "Python.h is not there"
    if missing:
        sys.stderr.write(f"{NATIVE.name} not built, for use from Python only: {missing}\n")
        return
    src = CSRC / "python" / "q3_native.cpp"
    newest = max(f.stat().st_mtime for f in (src, INCLUDE / "q3_ops.h", Path(torch.__file__)))
    if NATIVE.exists() and NATIVE.stat().st_mtime >= newest:
        return
    root = Path(torch.__file__).resolve().parent
    cuda = Path(shutil.which(NVCC) or "/usr/local/cuda/bin/nvcc").resolve().parent.parent
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={abi}", f"-I{INCLUDE}", f"-I{root}/include",
           f"-I{root}/include/torch/csrc/api/include", f"-I{sysconfig.get_paths()['include']}",
           f"-I{cuda}/include", str(src), "-o", str(NATIVE), f"-L{root}/lib", f"-L{lib.parent}",
           "-l:" + lib.name, "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda",
           "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{root}/lib"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"building {NATIVE.name} failed:\n{res.stdout}\n{res.stderr}")


def build(verbose: bool = False, clean: bool = False) -> Path:
    if clean and BUILD.exists():
        shutil.rmtree(BUILD)
    BUILD.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cpp"))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if LIB.exists() and all(LIB.stat().st_mtime >= o.stat().st_mtime for o in objs):
        _native(LIB)
        return LIB
    cmd = [NVCC, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", str(LIB), *map(str, objs),
           "-lcudart", "-lcuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    _native(LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--clean", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(verbose=a.verbose, clean=a.clean))
