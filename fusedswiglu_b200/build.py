"""Builds libfused_swiglu_sm100.so in-tree with nvcc for sm_100a.

Run as ``python -m fusedswiglu_b200.build`` (add ``--force`` to rebuild).  nvcc
cross-compiles without a GPU, so this also works on a CPU-only build machine.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_NAME = "libfused_swiglu_sm100.so"
LIB_PATH = PKG_DIR / LIB_NAME
SOURCES = [CSRC / "fsw_api.cu", CSRC / "fsw_route.cu", CSRC / "fsw_experts.cu", CSRC / "fsw_few.cu", CSRC / "fsw_fp8.cu"]
PUBLIC_HEADER = PKG_DIR.parent / "include" / "fused_swiglu.h"
HEADERS = [CSRC / "fsw_ptx.cuh", CSRC / "fsw_gemm.cuh", CSRC / "fsw_host.h", CSRC / "fsw_experts.h", PUBLIC_HEADER]
OBJ_DIR = CSRC / "build"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def find_nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or add it to PATH")
    return cand


def is_stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    return any(p.stat().st_mtime > built for p in SOURCES + HEADERS)


def _run(cmd) -> subprocess.CompletedProcess:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    return proc


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the shared library if it is missing or older than its sources: one object
    per source, in parallel, then one link."""
    if not force and not is_stale():
        return LIB_PATH
    nvcc = find_nvcc()
    OBJ_DIR.mkdir(exist_ok=True)
    newest_header = max(p.stat().st_mtime for p in HEADERS)
    objects, jobs = [], []
    for src in SOURCES:
        obj = OBJ_DIR / (src.stem + ".o")
        objects.append(obj)
        fresh = obj.exists() and obj.stat().st_mtime > max(newest_header, src.stat().st_mtime)
        if force or not fresh:
            jobs.append([nvcc, *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-c", "-o", str(obj), str(src)])
    with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        for proc in pool.map(_run, jobs):
            if verbose:
                sys.stderr.write(proc.stderr)
    tmp = LIB_PATH.with_suffix(".so.tmp")
    _run([nvcc, *NVCC_FLAGS, "-shared", "-o", str(tmp), *map(str, objects)])
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
