"""Build libmssample.so in place with nvcc for sm_100a (B200).

    python -m miniserve_b200.build

The library is a plain C-ABI shared object (no torch types in its
signatures); it links the CUDA runtime statically so it does not depend on
which libcudart the host process loaded.  _binding.so, beside it, holds the
Python entry points of the decode-step operators (csrc/ms_binding.cpp).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmssample.so")
BINDING = os.path.join(HERE, "_binding.so")
SOURCES = ["ms_sample.cu", "ms_kv.cu", "ms_attn.cu", "ms_int8.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libmssample.so")
    return path


def build(verbose: bool = False, extra_flags=None) -> str:
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(os.path.dirname(HERE), "include", "mssample.h"))
    if os.path.exists(LIB) and not extra_flags:
        lib_m = os.path.getmtime(LIB)
        if all(os.path.getmtime(d) <= lib_m for d in deps):
            return LIB
    cmd = [nvcc(), *ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", "-t", "0",
           "-Xptxas", "-v" if verbose else "-O3", "-o", LIB + ".tmp",
           *[os.path.join(CSRC, s) for s in SOURCES], *(extra_flags or [])]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    if verbose:
        sys.stdout.write(res.stdout + res.stderr)
    os.replace(LIB + ".tmp", LIB)
    return LIB


def build_binding() -> str:
    """Compile the Python entry points of the decode-step operators against
    the installed torch's headers; its libraries are those torch has loaded."""
    source = os.path.join(CSRC, "ms_binding.cpp")
    header = os.path.join(os.path.dirname(HERE), "include", "mssample.h")
    import torch
    root = os.path.dirname(torch.__file__)
    if os.path.exists(BINDING):
        made = os.path.getmtime(BINDING)
        if all(os.path.getmtime(d) <= made for d in (source, header, os.path.join(root, "version.py"))):
            return BINDING
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(root, "include"),
           "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"), "-isystem", cuda,
           source, "-o", BINDING + ".tmp", "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10",
           "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("g++ failed:\n" + res.stdout + res.stderr)
    os.replace(BINDING + ".tmp", BINDING)
    return BINDING


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
    print(build_binding())
