"""Builds ``libcrystalformer_b200.so`` in-tree with nvcc for sm_100a (cross-compiles without a GPU), and ``_torch_ops.so``, the torch
functions around part of it, with the host compiler.

    python -m crystalformer_b200.build [--verbose]

Each is rebuilt only when a source is newer than the existing binary.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
LIB_PATH = os.path.join(PKG, "libcrystalformer_b200.so")
SOURCES = sorted(glob.glob(os.path.join(PKG, "csrc", "*.cu")))
HEADERS = sorted(glob.glob(os.path.join(PKG, "csrc", "*.cuh"))) + [os.path.join(ROOT, "include", "crystalformer_b200.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "--std=c++17",
    "-Xcompiler", "-fPIC", "-shared", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(PKG, "csrc"),
]


BINDING_SOURCE, BINDING_PATH = os.path.join(PKG, "csrc", "torch_binding.cpp"), os.path.join(PKG, "_torch_ops.so")


def newer(target: str, sources) -> bool:
    if not os.path.exists(target):
        return False
    built = os.path.getmtime(target)
    return all(os.path.getmtime(f) <= built for f in sources)


def up_to_date() -> bool:
    return newer(LIB_PATH, SOURCES + HEADERS + [os.path.abspath(__file__)])


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """``_torch_ops.so``, which loads the library from its own folder."""
    if not force and newer(BINDING_PATH, [BINDING_SOURCE, HEADERS[-1], os.path.abspath(__file__)]):
        return BINDING_PATH
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    includes = [os.path.join(ROOT, "include"), os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    # (the system's compiler, as for the library: one that links its own C++ runtime in breaks streams and exceptions that cross torch's)
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_torch_ops",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *("-I" + i for i in includes), BINDING_SOURCE, "-o", BINDING_PATH,
           "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-L" + PKG, "-l:libcrystalformer_b200.so",
           "-Wl,-rpath,$ORIGIN"]
    env = dict(os.environ, PATH="/usr/bin:" + os.environ.get("PATH", ""))
    cmd[0] = shutil.which("g++", path=env["PATH"]) or "g++"
    proc = subprocess.run(cmd, capture_output=True, text=True, env=env)
    if verbose:
        sys.stderr.write(proc.stderr)
    if proc.returncode != 0:
        raise RuntimeError("building the torch functions failed:\n" + proc.stdout + proc.stderr)
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False) -> str:
    build_library(force, verbose)
    build_binding(force, verbose)
    return LIB_PATH


def build_library(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB_PATH
    nvcc = os.environ.get("NVCC", "nvcc")
    cmd = [nvcc, "--threads", "0"] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + SOURCES + ["-o", LIB_PATH]
    env = dict(os.environ)
    # the host compiler must be the system gcc
    env["PATH"] = "/usr/bin:" + env.get("PATH", "")
    proc = subprocess.run(cmd, capture_output=True, text=True, env=env)
    if verbose:
        sys.stderr.write(proc.stderr)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force=True, verbose="--verbose" in sys.argv))
