"""Build librbq.so (the C-ABI CUDA library) in-tree for sm_100a, and librbq_torch.so (PyTorch operators
over it) beside it.

Usage: ``python -m neurosamble_b200.build_ext`` (or ``build()`` from Python).  The shared
library lands in ``neurosamble_b200/_lib/librbq.so`` so it travels with the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(OUT_DIR, "librbq.so")
TORCH_LIB = os.path.join(OUT_DIR, "librbq_torch.so")
TORCH_VERSION = TORCH_LIB + ".torch"  # the version of torch that it was compiled against

SOURCES = ["rbq_host_math.cpp", "rbq_build.cu", "rbq_search.cu", "rbq_coarse_tc.cu", "rbq_gemm.cu", "rbq_norm.cu",
           "rbq_capi.cu"]
TORCH_SOURCE = "rbq_torch.cpp"  # PyTorch operators over the C ABI; a library of its own, so that C users need no torch
HEADERS = ["rbq_internal.cuh", "rbq_tc.cuh", os.path.join("..", "..", "include", "rbq.h")]

# -fmad=false: no FMA contraction anywhere, so every expression is evaluated as written and
# the results match the CPU oracle bit for bit.  IEEE division / sqrt stay on (no fast math).
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17", "-fmad=false",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-ffp-contract=off,-O3",
    "-Xptxas", "-warn-spills",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _cxx() -> str:
    for cand in ("/usr/bin/g++", shutil.which("g++")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("g++ not found")


def _environment() -> dict:
    env = dict(os.environ)
    env.pop("CXX", None)
    env.pop("CC", None)
    return env


def torch_version() -> str:
    """The running torch's version, "" without torch."""
    try:
        import torch
    except ImportError:
        return ""
    return str(torch.__version__)


def build_torch() -> None:
    """Compile the PyTorch operators against the running torch's headers and link them to librbq.so beside them."""
    import torch
    root = os.path.dirname(torch.__file__)
    include = os.path.join(root, "include")
    tmp = TORCH_LIB + ".tmp"
    subprocess.run([_cxx(), "-std=c++17", "-O2", "-fPIC", "-shared",
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + include,
                    "-I" + os.path.join(include, "torch", "csrc", "api", "include"), "-I/usr/local/cuda/include",
                    os.path.join(CSRC, TORCH_SOURCE), "-o", tmp, "-L" + os.path.join(root, "lib"), "-L" + OUT_DIR,
                    "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-lrbq", "-Wl,-rpath,$ORIGIN"],
                   check=True, env=_environment())
    if os.path.exists(TORCH_VERSION):  # never beside a library of another version
        os.remove(TORCH_VERSION)
    os.replace(tmp, TORCH_LIB)
    with open(TORCH_VERSION, "w") as f:
        f.write(torch_version() + "\n")


def _older(path: str, sources) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(os.path.join(CSRC, f)) > t for f in sources)


def _stale() -> bool:
    return _older(LIB, SOURCES + HEADERS)


def _torch_stale() -> bool:
    """librbq_torch.so is older than its sources, or was compiled against another torch than the running one."""
    if _older(TORCH_LIB, [TORCH_SOURCE, HEADERS[-1]]) or not os.path.exists(TORCH_VERSION):
        return True
    with open(TORCH_VERSION) as f:
        return f.read().strip() != torch_version()


def build(force: bool = False, verbose: bool = False) -> str:
    """Build what is out of date.  Without torch librbq.so is built alone: C users need no more."""
    if force or _stale():
        build_library(verbose)
    if torch_version() and (force or _torch_stale()):
        build_torch()
    return LIB


def build_library(verbose: bool = False) -> None:
    os.makedirs(OUT_DIR, exist_ok=True)
    nvcc = _nvcc()
    env = _environment()

    def compile_one(src: str) -> str:
        obj = os.path.join(OUT_DIR, os.path.splitext(src)[0] + ".o")
        extra = os.environ.get("RBQ_NVCC_EXTRA", "").split()
        cmd = [nvcc, *NVCC_FLAGS, *extra, "-c", os.path.join(CSRC, src), "-o", obj]
        if src.endswith(".cpp"):
            cmd = [_cxx(), "-std=c++17", "-O3", "-fPIC", "-ffp-contract=off", "-fno-fast-math",
                   "-I/usr/local/cuda/include", "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True, env=env)
        return obj

    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, SOURCES))
    tmp = LIB + ".tmp"
    # Static CUDA runtime: the library does not bind to whichever libcudart the host process
    # (e.g. PyTorch) loaded first; device pointers and streams are shared through the driver.
    cmd = [nvcc, "-shared", "-cudart=static", "-gencode", "arch=compute_100a,code=sm_100a", "-o", tmp, *objs]
    subprocess.run(cmd, check=True, env=env)
    os.replace(tmp, LIB)
    for o in objs:
        os.remove(o)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
