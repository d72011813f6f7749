"""Builds libcvn_hip.so (all HIP kernels + the C ABI of include/converse2d.h) for gfx950, in-tree.

Usage: python -m conversenet_amd.build   (or conversenet_amd.build.build()).  Each .hip source is
compiled to an object in parallel, then linked into conversenet_amd/lib/libcvn_hip.so.  Beside it comes
libcvn_autograd.so: host code against the installed torch's C++ interface (csrc/autograd_stream.cpp).
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "lib", "obj")
LIB = os.path.join(PKG, "lib", "libcvn_hip.so")
AUTOGRAD_LIB = os.path.join(PKG, "lib", "libcvn_autograd.so")
ARCH = os.environ.get("CVN_OFFLOAD_ARCH", "gfx950")

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
FLAGS = [
    "-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}",
    # packed fp32 VALU ops stay disabled on this target: some of their forms have given wrong results
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _compile(src: str) -> str:
    obj = os.path.join(OBJ, os.path.basename(src)[:-4] + ".o")
    cmd = [HIPCC, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def _build_autograd() -> str:
    import torch

    root = os.path.dirname(os.path.abspath(torch.__file__))
    cxx = shutil.which(os.environ.get("CXX", "g++")) or "/opt/rocm/llvm/bin/clang++"
    tmp = AUTOGRAD_LIB + ".tmp"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", os.path.join(root, "include"), "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-isystem", sysconfig.get_path("include"), os.path.join(CSRC, "autograd_stream.cpp"),
           "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cxx} failed for autograd_stream.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, AUTOGRAD_LIB)
    return AUTOGRAD_LIB


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        host = ex.submit(_build_autograd)
        objs = list(ex.map(_compile, srcs))
        host.result()
    tmp = LIB + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print("built", LIB)
        print("built", AUTOGRAD_LIB)
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
