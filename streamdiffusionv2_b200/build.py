"""Builds libsdv2.so (the CUDA kernels and their C ABI) in-tree with nvcc for sm_100a, and _calls.so, the PyTorch binding
of its newer entry points.

    python -m streamdiffusionv2_b200.build
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libsdv2.so")
CALLS = os.path.join(HERE, "_calls.so")
CALLS_SOURCE = os.path.join(CSRC, "torch_calls.cpp")
SOURCES = ["api.cu", "rope_append.cu", "attn_simt.cu", "attn_tcgen05.cu", "noalloc.cu", "block_elementwise.cu", "ring_plan.cu",
           "q8_cache.cu", "attn_q8_spans.cu", "attn_q8_few.cu"]
HEADERS = ["ptx.cuh", "attn_items.cuh", "attn_tiles.cuh", "rope_append.cuh", "q8.cuh", "sdv2_internal.h",
           os.path.join("..", "..", "include", "sdv2.h")]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or install the CUDA toolkit")


def sources():
    return [os.path.join(CSRC, s) for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]


def is_stale() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(CALLS):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(CALLS))
    deps = sources() + [CALLS_SOURCE] + [os.path.normpath(os.path.join(CSRC, h)) for h in HEADERS]
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def _calls_command():
    """The PyTorch binding of the newer entry points (a plain C++ extension module, no CUDA code)."""
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    lib = os.path.join(root, "lib")
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             "-o", CALLS, CALLS_SOURCE] + [f"-I{i}" for i in inc]
            + [f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"])


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu under csrc/ into libsdv2.so and the PyTorch binding into _calls.so; returns the library path."""
    if not force and not is_stale():
        return LIB
    cmd = [_nvcc(), "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
           "-Xcompiler", "-fPIC", "-shared", "-o", LIB] + sources()
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    binding = subprocess.Popen(_calls_command(), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    said, _ = binding.communicate()
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    if binding.returncode != 0:
        raise RuntimeError("g++ failed:\n" + said)
    if verbose:
        print(res.stdout + res.stderr + said)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose="-v" in sys.argv))
