"""Build the sm_100a shared library ``lib/libee_b200.so`` from ``csrc/`` with nvcc, and the extension module
``lib/ee_torch.so`` (the native host side of the prompt-layer operators) with g++.

The library is built in-tree so that it travels with the source checkout;
``python -m embodied_efficiency_b200.build`` (or ``__graft_entry__.build()``)
rebuilds it when any source is newer than the library, and the extension also
when it was built for another torch. The library needs nvcc alone; where the
extension cannot be built (no torch, its headers or g++), a warning says so and
the operators take the interpreter's path to the same kernels.
"""
from __future__ import annotations

import importlib.metadata
import os
import subprocess
import sys
import warnings
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


def _newer(target: str, files: list) -> bool:
    """``target`` is there and none of its sources is newer."""
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(f) <= t for f in files)


def up_to_date() -> bool:
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    files.remove(TORCH_SRC)
    return _newer(LIB, files + [os.path.join(INCLUDE, "ee_b200.h"), os.path.abspath(__file__)])


def torch_version() -> str:
    """The installed torch and the interpreter, which the extension is built for; empty without torch."""
    try:
        return f"{importlib.metadata.version('torch')} {sys.implementation.cache_tag}"
    except importlib.metadata.PackageNotFoundError:
        return ""


def _stamp() -> str:
    return os.path.join(os.path.dirname(TORCH_LIB), "obj", "ee_torch.version")


def torch_up_to_date() -> bool:
    if not _newer(TORCH_LIB, [TORCH_SRC, os.path.join(INCLUDE, "ee_b200.h"), os.path.abspath(__file__)]):
        return False
    try:
        with open(_stamp()) as f:
            return f.read() == torch_version()
    except OSError:
        return False


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
           f'-DEE_TORCH_VERSION="{torch_version()}"', TORCH_SRC, "-o", tmp, "-L", LIBDIR, "-l:libee_b200.so", "-L", os.path.join(tdir, "lib"), "-ltorch_python",
           "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {TORCH_SRC}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    os.makedirs(os.path.dirname(_stamp()), exist_ok=True)
    with open(_stamp(), "w") as f:
        f.write(torch_version())
    return TORCH_LIB


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    if force or not up_to_date():
        _build_lib(verbose, ptxas_info)
    if force or not torch_up_to_date():
        try:
            _build_torch()
        except (ImportError, OSError, RuntimeError) as e:
            warnings.warn(f"{TORCH_LIB} was not built, calls go through the interpreter: {e}", RuntimeWarning, stacklevel=2)
    return LIB


def _build_lib(verbose: bool, ptxas_info: bool):
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


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas" in sys.argv))
