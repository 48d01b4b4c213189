"""Builds libomni_moe_b200.so (the kernels, nvcc for sm_100a) and _binding.so (the torch binding of the short operators, g++)
in-tree; no GPU is needed to compile.

    python -m omni_moe_b200.build [--force] [--verbose]
"""
from __future__ import annotations

import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libomni_moe_b200.so")
BINDING = os.path.join(PKG, "_binding.so")
BINDING_SOURCE = os.path.join(CSRC, "binding.cpp")
SOURCES = ["capi.cu", "router_topk.cu", "schedule.cu", "expert.cu", "gemm_tcgen05.cu", "backward.cu", "elementwise.cu", "selftest.cu", "partition.cu", "decode.cu", "norm.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _deps():
    out = [os.path.join(CSRC, s) for s in SOURCES]
    out += [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    out.append(os.path.join(os.path.dirname(PKG), "include", "omni_moe_b200.h"))
    return out


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(d) > t for d in _deps())


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu file and link the shared library, then the torch binding; returns the library's path."""
    if not force and not needs_build():
        build_binding()
        return LIB
    objdir = os.path.join(PKG, "build")
    os.makedirs(objdir, exist_ok=True)
    procs = []
    for s in SOURCES:
        obj = os.path.join(objdir, s.replace(".cu", ".o"))
        cmd = [_nvcc(), *NVCC_FLAGS, "-c", os.path.join(CSRC, s), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        procs.append((s, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    objs = []
    for s, obj, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {s}:\n{out}")
        if verbose and out:
            print(out)
        objs.append(obj)
    link = [_nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB, *objs, "-lcudart"]
    r = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}")
    build_binding(force)
    return LIB


def binding_needs_build() -> bool:
    if not os.path.exists(BINDING):
        return True
    t = os.path.getmtime(BINDING)
    header = os.path.join(os.path.dirname(PKG), "include", "omni_moe_b200.h")
    return any(os.path.getmtime(d) > t for d in (BINDING_SOURCE, header))


def build_binding(force: bool = False) -> str:
    """Compile and link the torch binding against libomni_moe_b200.so (found next to it at run time); returns its path."""
    if not force and not binding_needs_build():
        return BINDING
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    include = [*cpp_extension.include_paths(), os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    libs = cpp_extension.library_paths()
    # the system compiler, not $CXX: one that links its own static libstdc++ breaks exceptions and streams inside torch's process
    gxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    cmd = [gxx, "-shared", "-fPIC", "-O2", "-std=c++17", "-fvisibility=hidden", "-w",
           "-DTORCH_EXTENSION_NAME=_binding", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{d}" for d in include), BINDING_SOURCE, "-o", BINDING, f"-L{PKG}", "-l:libomni_moe_b200.so",
           *(f"-L{d}" for d in libs), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN", *(f"-Wl,-rpath,{d}" for d in libs)]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on binding.cpp:\n{r.stdout}")
    return BINDING


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
