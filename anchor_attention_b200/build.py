"""Builds libanchor_attn_b200.so in-tree with nvcc for sm_100a, and the Python entry points of the
paged cache (_paged_binding.so) with the host compiler against it.

    python -m anchor_attention_b200.build [--force] [--verbose]

Without torch (the library alone): python anchor_attention_b200/build.py
"""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libanchor_attn_b200.so")
BINDING = os.path.join(HERE, "_paged_binding.so")
SOURCES = ["anchor_abi.cu", "paged_abi.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--expt-relaxed-constexpr", "-shared", "-Xcompiler", "-fPIC", "-cudart", "shared",
]


def _newest_source_mtime(endings=(".cu", ".cuh", ".h")):
    m = 0.0
    for root in (CSRC, os.path.join(HERE, "..", "include")):
        for f in os.listdir(root):
            if f.endswith(endings):
                m = max(m, os.path.getmtime(os.path.join(root, f)))
    return m


def _run(cmd, verbose, what):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"building {what} failed")


def build_library(force=False, verbose=False):
    """Compile the CUDA sources into the shared library and the Python binding of the paged cache against
    it; returns the library's path."""
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < _newest_source_mtime():
        nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
        _run([nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + [os.path.join(CSRC, s) for s in SOURCES] +
             ["-o", LIB], verbose, "libanchor_attn_b200.so")
    if force or not os.path.exists(BINDING) or os.path.getmtime(BINDING) < _newest_source_mtime((".cpp", ".h")):
        build_binding(verbose)
    return LIB


def build_binding(verbose=False):
    """Compile the Python entry points of the paged cache.  Where torch is missing there is nobody to call them: a user of the
    C interface has the library alone."""
    try:
        import torch
    except ImportError:
        sys.stderr.write("torch is not installed: _paged_binding.so is left out, the library is complete\n")
        return
    torch_dir = os.path.dirname(torch.__file__)
    include = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
               os.environ.get("CUDA_HOME", "/usr/local/cuda") + "/include", sysconfig.get_paths()["include"]]
    _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + ["-I" + d for d in include] +
         [os.path.join(CSRC, "paged_binding.cpp"), "-o", BINDING, "-L" + os.path.join(torch_dir, "lib"), "-ltorch",
          "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10", "-lc10_cuda", "-L" + HERE, "-l:libanchor_attn_b200.so",
          "-Wl,-rpath,$ORIGIN"], verbose, "_paged_binding.so")


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
