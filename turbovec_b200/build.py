"""Builds libturbovec_b200.so (CUDA kernels + host index + C ABI) for sm_100a with nvcc.

The library is built in-tree, next to this file.  `python -m turbovec_b200.build` rebuilds it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libturbovec_b200.so")
SOURCES = ["host_tables.cpp", "io_v7.cpp", "idtable.cpp", "multi.cpp", "ingest.cu", "ingest_fast.cu", "quantile.cu", "search.cu", "select.cu", "scan_lut.cu", "scan_filter.cu", "scan_small.cu", "scan_tc.cu", "scan_tc_wide.cu", "scan_tc_dense.cu", "scan_tc_dense2.cu", "kv_append.cu", "kv_attend.cu", "kv_prefix.cu", "kv_select.cu", "kv_api.cu", "index.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# -fmad=false: the reference never contracts a multiply and an add; fused operations are written
# explicitly (fmaf) where the reference has an explicit fma.
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-fmad=false", "-Xcompiler", "-fPIC,-ffp-contract=off,-O2",
              "--expt-relaxed-constexpr"]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build turbovec_b200")
    return path


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "turbovec_b200.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    procs = []
    for src in SOURCES:
        obj = os.path.join(objdir, src + ".o")
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode != 0:
            sys.stderr.write(out)
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}")
    subprocess.check_call([nvcc(), *ARCH, "-shared", "-o", LIB, *objs, "-lcudart"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
