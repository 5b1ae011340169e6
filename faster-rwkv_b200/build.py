"""Compile the sm_100a kernels and the C-ABI into csrc/libfr_b200.so, and the operators' torch entry into csrc/fr_b200_torch.so
(in-tree, nvcc and g++, no cmake).

nvcc cross-compiles without a GPU.  Object files are rebuilt only when a source or header is newer, the torch entry also when it was built for
another torch or Python.  Where there is no torch the library is built without that entry.
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import signal
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
LIB = os.path.join(CSRC, "libfr_b200.so")
TORCH_SOURCE = os.path.join(CSRC, "torch_ops.cpp")
TORCH_LIB = os.path.join(CSRC, "fr_b200_torch.so")
TORCH_STAMP = os.path.join(CSRC, "build", "torch_ops.txt")   # what TORCH_LIB was built for
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
    torch_build = _start_torch(force)
    try:
        _build_cuda(force, verbose, hdr)
    except BaseException:
        if torch_build is not None:
            os.killpg(torch_build.pid, signal.SIGTERM)   # (g++ and the compiler that it runs)
            torch_build.communicate()
        raise
    if torch_build is not None:
        out, _ = torch_build.communicate()
        if torch_build.returncode != 0:
            sys.stderr.write(out)
            raise RuntimeError("g++ failed on torch_ops.cpp")
        os.replace(TORCH_LIB + ".new", TORCH_LIB)
        with open(TORCH_STAMP, "w") as f:
            f.write(_torch_stamp())
    return LIB


def _build_cuda(force: bool, verbose: bool, hdr: float) -> None:
    objs, rebuilt = [], False
    procs = []
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


def _torch_stamp() -> str:
    """The torch and the Python that an extension is built for, without importing torch."""
    spec = importlib.util.find_spec("torch")
    return f"torch {importlib.metadata.version('torch')} at {spec.origin}, {sysconfig.get_config_var('SOABI')}\n"


def _start_torch(force: bool):
    """g++ on torch_ops.cpp, under way, or None where what is there is new enough, or where there is no torch to build it for."""
    if importlib.util.find_spec("torch") is None:
        sys.stderr.write("no torch: csrc/fr_b200_torch.so is not built (only the operators over torch tensors need it)\n")
        return None
    stamp = _torch_stamp()
    newest = max(os.path.getmtime(TORCH_SOURCE), os.path.getmtime(os.path.join(INCLUDE, "fr_b200.h")))
    if not force and os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) >= newest and os.path.exists(TORCH_STAMP):
        with open(TORCH_STAMP) as f:
            if f.read() == stamp:
                return None

    import torch
    base = os.path.dirname(torch.__file__)
    libs = os.path.join(base, "lib")
    cuda = os.environ.get("CUDA_HOME") or "/usr/local/cuda"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", os.path.join(base, "include"), "-I", os.path.join(base, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(cuda, "include"), TORCH_SOURCE, "-o", TORCH_LIB + ".new",
           "-L", libs, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", f"-Wl,-rpath,{libs}"]
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, start_new_session=True)


if __name__ == "__main__":
    print(build_lib(force="--force" in sys.argv, verbose=True))
