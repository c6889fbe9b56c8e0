"""Builds libwgblas_b200.so (the C ABI of include/wgblas.h) in-tree with nvcc for sm_100a.

Usage: python wgblas_b200/build.py [--force] [-v]   (runs without importing the package)
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libwgblas_b200.so")
BUILD_DIR = os.path.join(HERE, "_build")

SOURCES = ["runtime.cu", "gemm.cu", "gemm_simt.cu", "sgemm_tf32x3.cu", "sgemm_fused.cu", "probe.cu", "sgemm_noalloc.cu", "dgemm_dmma.cu", "shard.cu", "level3_aux.cu", "trsm.cu", "gemv.cu", "grouped.cu", "mx.cu"]
HEADERS = ["internal.h", "tcgen05.cuh", "tf32x3_common.cuh", "simt_tile.cuh", "grouped_common.cuh"]

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-ffp-contract=off",
         "--expt-relaxed-constexpr", "-I" + os.path.join(ROOT, "include")]


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD_DIR, exist_ok=True)
    headers = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(ROOT, "include", "wgblas.h")]
    objs, jobs = [], []
    for src in SOURCES:
        path = os.path.join(CSRC, src)
        obj = os.path.join(BUILD_DIR, src.replace(".cu", ".o"))
        objs.append(obj)
        if force or _stale(obj, [path] + headers):
            cmd = [NVCC, *ARCH, *FLAGS, "-c", path, "-o", obj]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)
    # The translation units compile independently: run them side by side.
    procs = [subprocess.Popen(cmd) for cmd in jobs]
    failed = [cmd for cmd, proc in zip(jobs, procs) if proc.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    if force or _stale(LIB, objs):
        subprocess.run([NVCC, *ARCH, "-shared", "-o", LIB, *objs, "-ldl"], check=True)
    build_napi(force)
    build_fast(force)
    return LIB


FAST_SRC = os.path.join(CSRC, "fastcall.c")
# (object slots are read by offset: the file is this interpreter's and no other's)
FAST = os.path.join(HERE, "_fast" + sysconfig.get_config_var("EXT_SUFFIX"))
PYTHON_INCLUDE = sysconfig.get_paths()["include"]


def build_fast(force: bool = False) -> str | None:
    """Builds the CPython extension _fast (csrc/fastcall.c) next to the library it calls. Without a C
    compiler or this interpreter's headers it is left out, and the package goes by its Python checks."""
    if not force and not _stale(FAST, [FAST_SRC, LIB, os.path.join(ROOT, "include", "wgblas.h")]):
        return FAST
    cc, header = shutil.which("gcc"), os.path.join(PYTHON_INCLUDE, "Python.h")
    if not cc or not os.path.exists(header) or sys.version_info < (3, 9):
        print("_fast (csrc/fastcall.c) is not built: it needs gcc, Python >= 3.9 and " + header, file=sys.stderr)
        return None
    subprocess.run([cc, "-std=c11", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    "-fvisibility=hidden", "-I" + os.path.join(ROOT, "include"), "-I" + PYTHON_INCLUDE, FAST_SRC,
                    "-L" + HERE, "-lwgblas_b200", "-Wl,-rpath,$ORIGIN", "-o", FAST], check=True)
    return FAST


NAPI_SRC = os.path.join(HERE, "napi", "wgblas_napi.c")
NAPI_ADDON = os.path.join(HERE, "napi", "wgblas_napi.node")
CUDA_HOME = os.path.dirname(os.path.dirname(NVCC))


def napi_command(out: str) -> list[str]:
    """gcc command line of the Node-API addon (Node resolves its napi_* symbols at load)."""
    return ["gcc", "-std=c11", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-fvisibility=hidden",
            "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(CUDA_HOME, "include"), NAPI_SRC,
            "-L" + HERE, "-lwgblas_b200", "-L" + os.path.join(CUDA_HOME, "lib64"), "-lcudart",
            "-Wl,-rpath,$ORIGIN/..", "-o", out]


def build_napi(force: bool = False) -> str:
    """Builds wgblas_napi.node next to its source (the JavaScript shim in napi/js loads it)."""
    if force or _stale(NAPI_ADDON, [NAPI_SRC, LIB, os.path.join(ROOT, "include", "wgblas.h")]):
        subprocess.run(napi_command(NAPI_ADDON), check=True)
    return NAPI_ADDON


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
