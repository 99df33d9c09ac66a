"""Build the sm_100a shared library ``lib/libee_b200.so`` from ``csrc/`` with nvcc, and the extension module
``lib/ee_torch.so`` (the native host side of the prompt-layer operators) with g++.

The library is built in-tree so that it travels with the source checkout;
``python -m embodied_efficiency_b200.build`` (or ``__graft_entry__.build()``)
rebuilds it when any source is newer than the library.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libee_b200.so")
TORCH_SRC = os.path.join(CSRC, "ee_torch.cpp")       # native host side of the prompt-layer operators
TORCH_LIB = os.path.join(LIBDIR, "ee_torch.so")      # a Python extension module linked against LIB
INCLUDE = os.path.join(os.path.dirname(PKG), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
                     "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def sources() -> list:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps() -> list:
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    files.append(os.path.join(INCLUDE, "ee_b200.h"))
    files.append(os.path.abspath(__file__))
    return files


def up_to_date() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(TORCH_LIB):
        return False
    t = min(os.path.getmtime(LIB), os.path.getmtime(TORCH_LIB))
    return all(os.path.getmtime(f) <= t for f in _deps())


def _build_torch() -> str:
    """Compile ``TORCH_SRC`` with g++ against this interpreter's torch."""
    import sysconfig

    import torch
    tdir = os.path.join(os.path.dirname(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(nvcc())) if os.path.sep in nvcc() else "/usr/local/cuda"
    tmp = TORCH_LIB + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", os.path.join(tdir, "include"), "-isystem", os.path.join(tdir, "include/torch/csrc/api/include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda, "include"), "-I", INCLUDE,
           TORCH_SRC, "-o", tmp, "-L", LIBDIR, "-l:libee_b200.so", "-L", os.path.join(tdir, "lib"), "-ltorch_python",
           "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {TORCH_SRC}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(LIBDIR, exist_ok=True)
    objdir = os.path.join(LIBDIR, "obj")
    os.makedirs(objdir, exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas_info else []

    def compile_one(src):
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        cmd = [nvcc()] + NVCC_FLAGS + extra + ["-I", INCLUDE, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
        return obj, r.stderr

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, sources()))
    if verbose or ptxas_info:
        for _, log in results:
            if log:
                sys.stderr.write(log)
    tmp = LIB + ".tmp"
    cmd = [nvcc()] + ARCH + ["-shared", "-o", tmp] + [o for o, _ in results] + ["-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    _build_torch()
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv))
