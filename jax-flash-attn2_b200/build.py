"""Builds libfa2_b200.so (the C-ABI library with the sm_100a kernels) with nvcc and the Python binding of its operators
for language models (jax_flash_attn2/_fa2_native.so) with g++, both in-tree.

Usage: python build.py [--force] [--verbose]
The library is written beside this file, the binding into the package, so that both travel with the source tree.
"""
from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "build")
LIB_PATH = os.path.join(HERE, "libfa2_b200.so")
BINDING_SRC = os.path.join(HERE, "binding", "fa2_native.cpp")
BINDING_PATH = os.path.join(HERE, "jax_flash_attn2", "_fa2_native.so")
SOURCES = ["api.cu", "fwd_sm100.cu", "fwd256_sm100.cu", "fwd_combine.cu", "bwd_sm100.cu", "bwd256_sm100.cu",
           "fwd_scored64_sm100.cu", "fwd_scored128_sm100.cu", "fwd_scored256_sm100.cu",
           "bwd_scored64_sm100.cu", "bwd_scored128_sm100.cu", "bwd_scored256_sm100.cu", "document_layout.cu",
           "paged_plan.cu", "paged64_sm100.cu", "paged128_sm100.cu", "paged128_rows_sm100.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the library cannot be built")
    return exe


def _newest_input() -> float:
    paths = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    paths.append(os.path.join(HERE, "..", "include", "fa2_b200.h"))
    paths.append(os.path.join(HERE, "..", "include", "fa2_b200_debug.h"))
    paths.append(os.path.join(HERE, "..", "include", "fa2_b200_lm.h"))
    paths.append(os.path.abspath(__file__))
    return max(os.path.getmtime(p) for p in paths)


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
    cmd = [_nvcc(), *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{res.stdout}\n{res.stderr}")
    if verbose:
        sys.stderr.write(res.stderr)
    return obj


def build_binding(force: bool = False) -> str:
    """Compiles the binding against the installed torch; returns its path."""
    newest = max(os.path.getmtime(p) for p in (BINDING_SRC, os.path.join(HERE, "..", "include", "fa2_b200.h"),
                                               os.path.join(HERE, "..", "include", "fa2_b200_lm.h"), os.path.abspath(__file__)))
    if not force and os.path.exists(BINDING_PATH) and os.path.getmtime(BINDING_PATH) >= newest:
        return BINDING_PATH
    import sysconfig

    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *("-I" + d for d in include), BINDING_SRC,
           "-o", BINDING_PATH, "-L" + os.path.join(root, "lib"), "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10_cuda",
           "-ltorch_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {BINDING_SRC}:\n{res.stdout}\n{res.stderr}")
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles every kernel for sm_100a, links the shared library and builds the binding; returns the library's path."""
    with concurrent.futures.ThreadPoolExecutor(max_workers=1) as pool:
        binding = pool.submit(build_binding, force)
        path = _build_library(force, verbose)
        binding.result()
    return path


def _build_library(force: bool, verbose: bool) -> str:
    if not force and os.path.exists(LIB_PATH) and os.path.getmtime(LIB_PATH) >= _newest_input():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        objs = list(pool.map(lambda s: _compile(s, verbose), SOURCES))
    cmd = [_nvcc(), "-shared", "-o", LIB_PATH, *objs]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
