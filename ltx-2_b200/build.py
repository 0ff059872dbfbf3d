"""Build the sm_100a C-ABI library ``lib/libltxfp8.so`` with nvcc (in-tree).

The whole CUDA side is one translation unit (``csrc/ltxfp8.cu``), so the device
status word and the kernels share one module.  The library links the CUDA
runtime statically and reaches the driver's tensor-map encoder through
``cudaGetDriverEntryPointByVersion``; it needs no torch headers.

The tensor-level calls of the residual-path and training operators
(``csrc/torch_binding.cpp``) are a second library, ``lib/_ltxfp8_torch.so``: host code
only, compiled with g++ against torch's headers and linked to the first by a
relative path.

Usage:  python ltx-2_b200/build.py [--force] [--verbose]
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
SRC_DIR = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libltxfp8.so")
BINDING_PATH = os.path.join(LIB_DIR, "_ltxfp8_torch.so")
INCLUDE = os.path.join(REPO, "include")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "-diag-suppress", "550",
]


def _sources():
    files = [os.path.join(SRC_DIR, f) for f in sorted(os.listdir(SRC_DIR)) if f.endswith((".cu", ".cuh"))]
    files.append(os.path.join(INCLUDE, "ltxfp8.h"))
    return files


def _stale(target, sources) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(f) > t for f in sources)


def needs_build() -> bool:
    return _stale(LIB_PATH, _sources())


def build_binding(force: bool = False) -> str:
    import sys
    import sysconfig

    import torch

    src = os.path.join(SRC_DIR, "torch_binding.cpp")
    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    tmp = os.path.join(LIB_DIR, "_ltxfp8_torch.tmp.so")
    # The system's g++, not $CXX: a compiler that links its own libstdc++ statically puts a second
    # C++ runtime beside torch's, and an exception that crosses them ends the process.
    cmd = [
        "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f'-DLTXFP8_TORCH_VERSION="{torch.__version__}"',
        "-I" + INCLUDE, "-isystem", os.path.join(root, "include"),
        "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
        "-isystem", os.path.join(cuda, "include"), "-isystem", sysconfig.get_paths()["include"],
        src, "-o", tmp, "-L" + LIB_DIR, "-l:libltxfp8.so", "-L" + os.path.join(root, "lib"),
        "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    # What it was built with, beside it: file times do not tell that torch or Python has changed.
    # (Without the folders, which differ between machines that share the tree.)
    record = BINDING_PATH + ".built_with"
    key = f"torch {torch.__version__}, python {sys.version.split()[0]}, {' '.join(cmd[1:8])}"
    if not force and not _stale(BINDING_PATH, [src, os.path.join(INCLUDE, "ltxfp8.h")]) and os.path.exists(record):
        with open(record) as f:
            if f.read() == key:
                return BINDING_PATH
    subprocess.check_call(cmd)
    if b"libstdc++.so" not in subprocess.check_output(["readelf", "-d", tmp]):
        raise RuntimeError("the tensor-level binding must share torch's C++ runtime (libstdc++.so), but g++ linked its own")
    os.replace(tmp, BINDING_PATH)
    with open(record, "w") as f:
        f.write(key)
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        build_binding()
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    nvcc = os.environ.get("NVCC", "nvcc")
    if not os.path.isabs(nvcc) and os.path.exists("/usr/local/cuda/bin/nvcc"):
        nvcc = "/usr/local/cuda/bin/nvcc"
    cmd = [nvcc, *NVCC_FLAGS, "-I" + INCLUDE, "-o", LIB_PATH + ".tmp", os.path.join(SRC_DIR, "ltxfp8.cu")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd))
    subprocess.check_call(cmd)
    os.replace(LIB_PATH + ".tmp", LIB_PATH)
    build_binding(force)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(LIB_PATH)
