"""Build libl3dops.so (all CUDA kernels + the C ABI) for sm_100a with nvcc, and
_l3dpack.so (tensor descriptors for the Python front end) with the host compiler.

Objects are compiled in parallel into `_build/` beside this file and linked
into `libl3dops.so` in the package directory (in-tree, so the library travels
with the repository snapshot).  Rebuilds only what changed (source or shared
header newer than the object).
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.metadata
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libl3dops.so"
PACK = PKG / "_l3dpack.so"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", f"-I{ROOT / 'include'}", f"-I{CSRC}"]


def _sources():
    return sorted(CSRC.glob("*.cu"))


def _headers():
    return sorted(CSRC.glob("*.cuh")) + sorted((ROOT / "include").glob("*.h"))


def _needs(src: Path, obj: Path) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return src.stat().st_mtime > t or any(h.stat().st_mtime > t for h in _headers())


def _compile(src: Path) -> Path:
    obj = BUILD / (src.stem + ".o")
    if _needs(src, obj):
        cmd = [NVCC, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stderr}")
    return obj


def _pack_for() -> str:
    """What _l3dpack.so is bound to: the interpreter and the installed torch."""
    return f"{sysconfig.get_config_var('SOABI')} torch {importlib.metadata.version('torch')}"


def _pack_needs() -> bool:
    src, hdr, was = PKG / "host" / "pack.cpp", ROOT / "include" / "l3d_ops.h", BUILD / "_l3dpack.for"
    if not PACK.exists() or not was.exists() or was.read_text() != _pack_for():
        return True
    return PACK.stat().st_mtime <= max(src.stat().st_mtime, hdr.stat().st_mtime)


def _pack_module() -> None:
    """host/pack.cpp -> _l3dpack.so, against the headers of the installed torch."""
    if not _pack_needs():
        return
    import torch

    src = PKG / "host" / "pack.cpp"

    t = Path(torch.__file__).resolve().parent
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{ROOT / 'include'}",
           f"-isystem{t / 'include'}", f"-isystem{t / 'include/torch/csrc/api/include'}",
           f"-isystem{sysconfig.get_paths()['include']}", str(src), "-o", str(PACK), f"-L{t / 'lib'}",
           "-ltorch_python", "-ltorch_cpu", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{src.name} failed to compile:\n{r.stderr}")
    (BUILD / "_l3dpack.for").write_text(_pack_for())


def build(verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    if not LIB.exists() or any(o.stat().st_mtime > LIB.stat().st_mtime for o in objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    _pack_module()
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
