# -*- coding: utf-8 -*-
"""Build libptq8.so (sm_100a) in-tree with nvcc.

    python -m ptq_int8_lab_b200.build

The library is plain CUDA runtime + C++ (no torch linkage); the Python host
side loads it with ctypes.  Output: ptq_int8_lab_b200/_lib/libptq8.so, and
where torch is installed ptq8_host.so beside it, the Python extension that reads
torch tensors for the newer token operators' calls (C++ against torch's headers,
no CUDA).  The library does not depend on it, in its build or in its use.
"""
import os
import subprocess
import sys
import sysconfig
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
    ("ptq8_cache.cu", "ptq8_cache.o", ["-lineinfo"]),
    ("ptq8_w4.cu", "ptq8_w4.o", ["-lineinfo"]),
)


HOST = OUT / "ptq8_host.so"


def host_command(out: Path) -> list:
    """The compiler's command for ptq8_host.so; empty where there is no torch to read tensors of."""
    try:
        import torch
    except ImportError:
        return []
    root = Path(torch.__file__).resolve().parent
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-I", str(HERE.parent / "include"),
            "-I", sysconfig.get_paths()["include"], "-I", str(root / "include"), "-I", str(root / "include/torch/csrc/api/include"),
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", str(SRC / "ptq8_host.cpp"), "-o", str(out),
            "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]


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
    host_tmp = OUT / "ptq8_host.so.tmp"
    host_cmd, host = host_command(host_tmp), None
    if host_cmd:
        print(" ".join(host_cmd), flush=True)
        host = subprocess.Popen(host_cmd)
    else:
        print("no torch: libptq8.so alone, without ptq8_host.so", flush=True)
    failed = [cmd for cmd, p in running if p.wait() != 0]
    host_failed = host is not None and host.wait() != 0
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    tmp = OUT / "libptq8.so.tmp"
    cmd = [NVCC, "-shared", *ARCH, *[str(o) for o in objs], "-o", str(tmp), "-lcudart"]
    print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, lib)
    for o in objs:
        o.unlink()
    if host_failed:   # (libptq8.so is there, and all that does not need the extension works)
        raise subprocess.CalledProcessError(1, host_cmd)
    if host is not None:
        os.replace(host_tmp, HOST)
    return lib


if __name__ == "__main__":
    build(verbose_ptxas="-v" in sys.argv)
