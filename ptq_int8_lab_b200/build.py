# -*- coding: utf-8 -*-
"""Build libptq8.so (sm_100a) in-tree with nvcc.

    python -m ptq_int8_lab_b200.build

The library is plain CUDA runtime + C++ (no torch linkage); the Python host
side loads it with ctypes.  Output: ptq_int8_lab_b200/_lib/libptq8.so.
"""
import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
SRC = HERE / "csrc"
OUT = HERE / "_lib"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


# (source, object, further nvcc flags)
SOURCES = (
    ("ptq8_model.cpp", "ptq8_model.o", ["-x", "c++"]),
    ("ptq8_engine.cu", "ptq8_engine.o", ["-lineinfo"]),
    ("ptq8_ops.cu", "ptq8_ops.o", ["-lineinfo"]),
)


def build(verbose_ptxas: bool = False) -> Path:
    OUT.mkdir(exist_ok=True)
    lib = OUT / "libptq8.so"
    common = ["-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-I", str(HERE.parent / "include"), *ARCH]
    objs, running = [], []
    for src, obj, flags in SOURCES:      # one compiler process per source, side by side
        extra = ["-Xptxas", "-v"] if verbose_ptxas and src.endswith(".cu") else []
        cmd = [NVCC, *common, *flags, *extra, "-c", str(SRC / src), "-o", str(OUT / obj)]
        print(" ".join(cmd), flush=True)
        objs.append(OUT / obj)
        running.append((cmd, subprocess.Popen(cmd)))
    failed = [cmd for cmd, p in running if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    tmp = OUT / "libptq8.so.tmp"
    cmd = [NVCC, "-shared", *ARCH, *[str(o) for o in objs], "-o", str(tmp), "-lcudart"]
    print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, lib)
    for o in objs:
        o.unlink()
    return lib


if __name__ == "__main__":
    build(verbose_ptxas="-v" in sys.argv)
