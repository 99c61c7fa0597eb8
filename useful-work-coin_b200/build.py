"""Build libuwcb200.so (the C-ABI library) for sm_100a with nvcc, in-tree.

    python useful-work-coin_b200/build.py [--force] [--verbose]

Output: useful-work-coin_b200/uwc_b200/libuwcb200.so, linked against the static CUDA runtime so
it loads on a machine without a GPU driver (the symbol-export test runs on CPU-only hosts), and beside
it _paged.so, the torch side of uwc_b200.paged (C++, no device code), linked to it and to torch (where
there is a CUDA build of torch).
Nothing is compiled at import time: the product path refuses to run without this library.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "uwc_b200", "libuwcb200.so")
SOURCES = ["host.cu", "prep.cu", "gemm_sm100.cu", "mined.cu", "peak.cu", "stream_gemm.cu", "tp.cu", "detq.cu", "attn.cu", "sha.cu",
           "paged.cu", "paged_attn.cu", "paged_tile.cu"]
HEADERS = ["uwc_device.cuh", "uwc_host.h", "det_math.cuh", "uwc_tp.cuh", "paged.cuh"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
              "-Xcompiler", "-fPIC", "-cudart", "static"]


def nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else shutil.which("nvcc") or "nvcc"


EXT_SOURCE = "paged_torch.cpp"
EXT_OUT = os.path.join(HERE, "uwc_b200", "_paged.so")
EXT_STAMP = os.path.join(HERE, "_build", "paged_torch.stamp")   # the torch and the Python that it was built for


def build_extension(force: bool = False, verbose: bool = False) -> str | None:
    """The torch extension module: calls of the library from tensors. None where there is no CUDA torch to build it
    for: the library, for C callers and the ctypes modules, needs nvcc alone."""
    try:
        import torch
        found = torch.version.cuda is not None
    except ImportError:
        found = False
    if not found:
        print(f"{os.path.basename(EXT_OUT)} is not built: no CUDA build of torch here (only uwc_b200.paged and .serve need it)",
              file=sys.stderr)
        return None
    src = os.path.join(CSRC, EXT_SOURCE)
    inputs = [src, os.path.join(ROOT, "include", "uwc_b200.h")]
    stamp = f"{torch.__version__} {os.path.dirname(torch.__file__)} {sys.version}"
    if (not force and os.path.exists(EXT_OUT) and all(os.path.getmtime(f) <= os.path.getmtime(EXT_OUT) for f in inputs)
            and os.path.exists(EXT_STAMP) and open(EXT_STAMP).read() == stamp):
        return EXT_OUT
    import sysconfig

    from torch.utils import cpp_extension
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], *[d for d in [cuda] if d != "/usr/include"]]
    libdir = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = EXT_OUT + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[f"-isystem{d}" for d in includes], src, "-o", tmp, f"-L{libdir}", f"-Wl,-rpath,{libdir}", "-Wl,-rpath,$ORIGIN",
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", OUT]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, EXT_OUT)
    os.makedirs(os.path.dirname(EXT_STAMP), exist_ok=True)
    with open(EXT_STAMP, "w") as f:
        f.write(stamp)
    return EXT_OUT


def _inputs():
    files = [os.path.join(CSRC, f) for f in SOURCES + HEADERS]
    files.append(os.path.join(ROOT, "include", "uwc_b200.h"))
    return files


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(f) <= t for f in _inputs())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        build_extension(force, verbose)
        return OUT
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    for src in SOURCES:
        obj = os.path.join(objdir, src.replace(".cu", ".o"))
        cmd = [nvcc(), *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        objs.append(obj)
    tmp = OUT + ".tmp"
    subprocess.check_call([nvcc(), "-shared", "-cudart", "static", "-gencode", "arch=compute_100a,code=sm_100a",
                           "-Xlinker", "-soname=libuwcb200.so", *objs, "-o", tmp])
    os.replace(tmp, OUT)
    build_extension(force, verbose)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    sys.exit(0)
