"""Build the sm_100a shared library ``libthetascan_b200.so`` in-tree with nvcc.

The library is one translation unit (``csrc/all.cu``) exposing the C ABI of
``include/thetascan_b200.h``.  It is rebuilt when any source or the header is
newer than the library.  ``_host.so`` beside it is the Python extension
``csrc/host.cpp`` over that ABI (the host side of the operators whose calls are
short), built with the host compiler against the installed PyTorch.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libthetascan_b200.so")
HOST = os.path.join(HERE, "_host.so")
HOST_SOURCE = os.path.join(HERE, "csrc", "host.cpp")
HEADER = os.path.join(ROOT, "include", "thetascan_b200.h")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _sources():
    return [s for s in sorted(glob.glob(os.path.join(HERE, "csrc", "*"))) if s != HOST_SOURCE] + [HEADER]


def _stale(output, sources) -> bool:
    return not os.path.exists(output) or any(os.path.getmtime(s) > os.path.getmtime(output) for s in sources)


def needs_build() -> bool:
    return _stale(LIB, _sources())


def nvcc_command(output: str = LIB, extra=()) -> list[str]:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return [nvcc, *ARCH, "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
            "-Xcompiler", "-fPIC", "-shared", "-I", os.path.join(ROOT, "include"),
            *extra, "-o", output, os.path.join(HERE, "csrc", "all.cu")]


def host_command(output: str = HOST) -> list[str]:
    import torch
    at, cuda = torch.__path__[0], os.path.dirname(os.path.dirname(os.path.realpath(nvcc_command()[0])))
    includes = [f"-I{p}" for p in (f"{at}/include", f"{at}/include/torch/csrc/api/include", f"{cuda}/include",
                                   sysconfig.get_paths()["include"])]
    libraries = [f"-L{at}/lib", f"-L{cuda}/lib64"]
    return [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *includes, "-o", output, HOST_SOURCE,
            *libraries, f"-L{HERE}", "-l:libthetascan_b200.so", "-Wl,-rpath,$ORIGIN",
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-lcudart"]


def build_host(force: bool = False, verbose: bool = False) -> str:
    """Compile the Python extension if it is missing or stale; return its path."""
    if force or _stale(HOST, [HOST_SOURCE, HEADER]):
        cmd = host_command(HOST + ".tmp")
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
        os.replace(HOST + ".tmp", HOST)
    return HOST


def build(force: bool = False, verbose: bool = False, extra=()) -> str:
    """Compile the library and the extension where missing or stale; return the library's path."""
    if force or needs_build():
        cmd = nvcc_command(extra=extra)
        if verbose:
            print(" ".join(cmd))
        tmp = LIB + ".tmp"
        cmd[cmd.index(LIB)] = tmp
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB)
    build_host(force, verbose)
    return LIB


if __name__ == "__main__":
    build(force=True, verbose=True)
