"""Build ``libleanselect_b200.so`` (sm_100a) in-tree with nvcc.

Usage: ``python -m leanselect_b200.build [--force] [--verbose]``.

The library lands in ``leanselect_b200/_lib`` next to the sources so that it
travels with a copy of the repository.  The CUDA runtime is linked
statically: the library then does not depend on which ``libcudart`` the
host process (PyTorch) loaded first.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "libleanselect_b200.so"
# The compiled Python entry of the paged-cache operators; it is built against
# the installed torch, whose version its stamp file records.
BINDING = LIB_DIR / "_binding.so"
BINDING_STAMP = LIB_DIR / "_binding.torch"
BINDING_SOURCE = CSRC / "binding.cpp"
SOURCES = ["prep.cu", "score_select.cu", "sparse_attn.cu", "capi.cu", "backbone.cu", "noalloc.cu",
           "waitprobe.cu", "select_f32.cu", "paged_cache.cu", "paged_attn.cu"]
HEADERS = ["common.cuh", "launch.h", "topk_rows.cuh", "page_list.cuh", "paged_schedule.h"]

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists() and shutil.which(cand) is None:
        raise RuntimeError("nvcc not found; set NVCC or put CUDA 12.8+ on PATH")
    return cand


def _stale() -> bool:
    if not LIB.exists():
        return True
    built = LIB.stat().st_mtime
    inputs = [CSRC / s for s in SOURCES + HEADERS] + sorted((ROOT / "include").glob("*.h")) + [
        Path(__file__)]
    return any(p.stat().st_mtime > built for p in inputs)


def _binding_stale(torch_version: str) -> bool:
    if not BINDING.exists() or not BINDING_STAMP.exists():
        return True
    if BINDING_STAMP.read_text() != torch_version:
        return True
    built = BINDING.stat().st_mtime
    inputs = [BINDING_SOURCE, ROOT / "include" / "leanselect_b200.h", Path(__file__)]
    return any(p.stat().st_mtime > built for p in inputs)


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile the Python entry module against the installed torch (host code only)."""
    import sysconfig

    import torch

    if not force and not _binding_stale(torch.__version__):
        return BINDING
    home = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", str(home / "include"),
           "-isystem", str(home / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(cuda / "include"),
           str(BINDING_SOURCE), "-o", str(tmp), f"-L{LIB_DIR}", f"-L{home / 'lib'}",
           "-lleanselect_b200", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    BINDING_STAMP.write_text(torch.__version__)
    return BINDING


def build(force: bool = False, verbose: bool = False, extra_flags=()) -> Path:
    """Compile every kernel for sm_100a, link the shared library and its Python entry."""
    if force or _stale():
        _build_library(verbose, extra_flags)
    build_binding(force, verbose)
    return LIB


def _build_library(verbose: bool, extra_flags) -> None:
    LIB_DIR.mkdir(exist_ok=True)
    obj_dir = LIB_DIR / "obj"
    obj_dir.mkdir(exist_ok=True)
    cc = nvcc()
    objects = []
    for src in SOURCES:
        obj = obj_dir / (Path(src).stem + ".o")
        cmd = [cc, *ARCH, *NVCC_FLAGS, *extra_flags, "-I", str(ROOT / "include"), "-c",
               str(CSRC / src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objects.append(str(obj))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *objects, "-lpthread",
           "-ldl", "-lrt"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print register/smem usage")
    args = ap.parse_args(argv)
    extra = ["-Xptxas", "-v"] if args.ptxas_info else []
    path = build(force=args.force or args.ptxas_info, verbose=args.verbose, extra_flags=extra)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
