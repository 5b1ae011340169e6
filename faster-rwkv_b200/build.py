"""Compile the sm_100a kernels and the C-ABI into csrc/libfr_b200.so, and the operators' torch entry into csrc/fr_b200_torch.so
(in-tree, nvcc and g++, no cmake).

nvcc cross-compiles without a GPU.  Object files are rebuilt only when a source or header is newer.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
LIB = os.path.join(CSRC, "libfr_b200.so")
TORCH_SOURCE = os.path.join(CSRC, "torch_ops.cpp")
TORCH_LIB = os.path.join(CSRC, "fr_b200_torch.so")
SOURCES = ["pack.cu", "decode.cu", "step.cu", "prefill.cu", "sample.cu", "api.cu", "noalloc.cu", "ops.cu", "recur.cu", "linear.cu",
           "ssm_f16.cu", "ssm_bf16.cu", "ssm_f32.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xptxas", "-v"]


def _newest_header() -> float:
    t = 0.0
    for d in (CSRC, INCLUDE):
        for f in os.listdir(d):
            if f.endswith((".h", ".cuh")):
                t = max(t, os.path.getmtime(os.path.join(d, f)))
    return t


def build_lib(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(os.path.join(CSRC, "build"), exist_ok=True)
    hdr = _newest_header()
    objs, rebuilt = [], False
    procs = []
    torch_build = _start_torch(force)
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        if not os.path.exists(s):
            continue
        o = os.path.join(CSRC, "build", src.replace(".cu", ".o"))
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr):
            cmd = ["nvcc", *ARCH, *FLAGS, "-I", INCLUDE, "-c", s, "-o", o]
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
            rebuilt = True
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode != 0:
            sys.stderr.write(out)
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}")
        with open(os.path.join(CSRC, "build", src.replace(".cu", ".ptxas.txt")), "w") as f:
            f.write(out)
    if rebuilt or not os.path.exists(LIB):
        subprocess.check_call(["nvcc", *ARCH, "-shared", "-o", LIB, *objs])
    if torch_build is not None:
        out, _ = torch_build.communicate()
        if torch_build.returncode != 0:
            sys.stderr.write(out)
            raise RuntimeError("g++ failed on torch_ops.cpp")
    return LIB


def _start_torch(force: bool):
    """g++ on torch_ops.cpp, under way, or None where what is there is new enough."""
    newest = max(os.path.getmtime(TORCH_SOURCE), os.path.getmtime(os.path.join(INCLUDE, "fr_b200.h")))
    if not force and os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) >= newest:
        return None
    import sysconfig

    import torch
    base = os.path.dirname(torch.__file__)
    libs = os.path.join(base, "lib")
    cuda = os.environ.get("CUDA_HOME") or "/usr/local/cuda"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", os.path.join(base, "include"), "-I", os.path.join(base, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(cuda, "include"), TORCH_SOURCE, "-o", TORCH_LIB,
           "-L", libs, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", f"-Wl,-rpath,{libs}"]
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


if __name__ == "__main__":
    print(build_lib(force="--force" in sys.argv, verbose=True))
