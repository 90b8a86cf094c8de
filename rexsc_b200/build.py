"""Build librexsc_b200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a, and _host.so (the Python extension for the
host's side of some calls) with the host compiler.

    python -m rexsc_b200.build [--force]

nvcc cross-compiles without a GPU; the shared objects are written next to this file so that they are
found by rexsc_b200._lib and travel with the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "librexsc_b200.so")
HOST = os.path.join(HERE, "_host.so")
HOST_SOURCE = "host.cpp"
SOURCES = ["capi.cu", "sc_stream.cu", "sc_conv_direct.cu", "sc_conv_tiled.cu", "pointwise.cu", "fxp_conv.cu",
           "sc_conv_static.cu", "fxp_conv_umma.cu", "sc_conv_tc.cu", "caller_fused.cu",
           "int8_quantize.cu", "int8_matmul.cu", "adamw.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared", "--threads", "0",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: cannot build librexsc_b200.so")


def _header() -> str:
    return os.path.join(os.path.dirname(HERE), "include", "rexsc_b200.h")


def _older(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def needs_build() -> bool:
    return _older(LIB, [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f != HOST_SOURCE] + [_header()])


def needs_host_build() -> bool:
    return _older(HOST, [os.path.join(CSRC, HOST_SOURCE), _header()])


def build_host() -> None:
    """_host.so: linked against torch and the CUDA library beside it."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    libs = cpp_extension.library_paths()
    # the system's compiler, whose C++ runtime the interpreter loads (a newer one named by CXX links code of its own runtime in)
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           "-DTORCH_EXTENSION_NAME=_host", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f for d in include for f in ("-isystem", d)], "-o", HOST, os.path.join(CSRC, HOST_SOURCE),
           *[f for d in libs for f in ("-L" + d, "-Wl,-rpath," + d)], "-L" + HERE, "-Wl,-rpath,$ORIGIN",
           "-l:librexsc_b200.so", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    subprocess.check_call(cmd, cwd=CSRC)


def build(force: bool = False, verbose: bool = False) -> str:
    if force or needs_build():
        cmd = [_nvcc(), *NVCC_FLAGS, "-o", LIB] + [os.path.join(CSRC, s) for s in SOURCES]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        subprocess.check_call(cmd, cwd=CSRC)
    if force or needs_host_build():
        build_host()
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
