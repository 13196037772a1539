"""Builds the in-tree shared library macrograd_b200/libmg_gemm.so for sm_100a.

    python -m macrograd_b200.build        (or build() from Python)

nvcc cross-compiles without a GPU. The library links the CUDA runtime
statically and reaches the driver's tensor-map encoder through
cudaGetDriverEntryPoint, so it needs no libcuda at link time.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
LIB = os.path.join(PKG, "libmg_gemm.so")
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "_build")
INCLUDE = os.path.join(ROOT, "include")
# translation unit -> what it includes
UNITS = {
    "mg_gemm.cu": ["mg_gemm_kernel.cuh", "mg_ptx.cuh", "mg_host.h", "mg_plan.h"],
    "mg_attention.cu": ["mg_attention_host.h", "mg_attention_common.cuh", "mg_attention_math.cuh",
                        "mg_attention_simt.cuh", "mg_attention_tc.cuh",
                        "mg_attention_tc_bwd.cuh", "mg_attention_tc32.cuh", "mg_attention_tc32_bwd.cuh", "mg_tc16.cuh",
                        "mg_ptx.cuh", "mg_host.h", "mg_overlap.h"],
    "mg_paged.cu": ["mg_attention_host.h", "mg_attention_common.cuh", "mg_attention_math.cuh", "mg_paged.cuh",
                    "mg_rotary.cuh", "mg_ptx.cuh", "mg_host.h", "mg_overlap.h"],
}
SOURCES = [os.path.join(CSRC, u) for u in UNITS]
HEADERS = [os.path.join(INCLUDE, h) for h in ("mg_gemm.h", "mg_attention.h")]
DEPS = SOURCES + sorted({os.path.join(CSRC, h) for hs in UNITS.values() for h in hs}) + HEADERS
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = os.path.join(home, "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in DEPS if os.path.exists(p))


def _object(unit: str, force: bool, verbose: bool) -> str:
    """Compiles one translation unit if it, or what it includes, is newer."""
    obj = os.path.join(OBJ, unit.replace(".cu", ".o"))
    needs = [os.path.join(CSRC, f) for f in [unit] + UNITS[unit]] + HEADERS
    if not force and os.path.exists(obj) and all(os.path.getmtime(p) <= os.path.getmtime(obj) for p in needs):
        return obj
    cmd = [nvcc(), *ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-I" + INCLUDE, "-c", "-o", obj,
           os.path.join(CSRC, unit)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(len(UNITS)) as pool:
        objs = list(pool.map(lambda u: _object(u, force, verbose), UNITS))
    subprocess.run([nvcc(), *ARCH, "-Xcompiler", "-fPIC", "-shared", "-o", LIB, *objs], check=True)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
