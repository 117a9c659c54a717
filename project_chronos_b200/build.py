"""Build the sm_100a extension in-tree: project_chronos_b200/libchronos_moe.so, and the
Python module project_chronos_b200/_binding.so that checks tensors and calls it.

    python -m project_chronos_b200.build [--force]

nvcc cross-compiles for sm_100a without a GPU; the library links the CUDA
runtime statically and reaches the driver API (cuTensorMapEncodeTiled)
through cudaGetDriverEntryPoint, so it needs no libcuda at link time.
"""
from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB = os.path.join(PKG, "libchronos_moe.so")
BINDING = os.path.join(PKG, "_binding.so")
BINDING_STAMP = BINDING + ".txt"   # what it was built against
OBJ = os.path.join(PKG, "_build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def headers():
    return sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")))


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(f) > t for f in sources() + headers())


def _binding_sources():
    return [os.path.join(CSRC, "binding.cpp")] + sorted(glob.glob(os.path.join(INCLUDE, "*.h")))


def binding_target() -> str:
    """What _binding.so has to fit: the interfaces of this Python and of this torch."""
    import torch
    return f"{sysconfig.get_config_var('SOABI')} torch {torch.__version__} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}"


def binding_fits(unknown: bool) -> bool:
    """Whether _binding.so was built against what runs now; `unknown` where nothing says so."""
    if not os.path.exists(BINDING_STAMP):
        return unknown
    with open(BINDING_STAMP) as f:
        return f.read() == binding_target()


def needs_binding() -> bool:
    if not os.path.exists(BINDING) or not binding_fits(unknown=False):
        return True
    t = os.path.getmtime(BINDING)
    return any(os.path.getmtime(f) > t for f in _binding_sources())


def _binding_command() -> list:
    """g++ against the headers and libraries of the torch that imports it; the library beside it."""
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-I", INCLUDE,
            "-isystem", os.path.join(root, "include"), "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
            "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda, "include"),
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", os.path.join(CSRC, "binding.cpp"), LIB,
            "-L", os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN",
            "-o", BINDING + ".tmp"]


def _up_to_date(obj: str) -> bool:
    """Whether the object is newer than every file nvcc read for it (its .d list)."""
    if not (os.path.exists(obj) and os.path.exists(obj + ".d")):
        return False
    with open(obj + ".d") as f:
        deps = f.read().replace("\\\n", " ").split(":", 1)[1].split()
    t = os.path.getmtime(obj)
    return all(os.path.exists(d) and os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if force or needs_build():
        _build_library(force, verbose)
    if force or needs_binding():
        cmd = _binding_command()
        if verbose:
            print(" ".join(cmd))
        subprocess.check_call(cmd)
        if os.path.exists(BINDING_STAMP):
            os.remove(BINDING_STAMP)
        os.replace(BINDING + ".tmp", BINDING)
        with open(BINDING_STAMP, "w") as f:
            f.write(binding_target())
    return LIB


def _build_library(force: bool, verbose: bool) -> None:
    # one object per translation unit, compiled side by side and linked into one library
    flags = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden", "-I", INCLUDE,
             "-I", CSRC, "--expt-relaxed-constexpr", "-cudart", "static"]
    if verbose:
        flags.append("-Xptxas=-v")
    os.makedirs(OBJ, exist_ok=True)
    objects, running = [], []
    for src in sources():
        obj = os.path.join(OBJ, os.path.basename(src) + ".o")
        objects.append(obj)
        if not force and _up_to_date(obj):
            continue
        cmd = [nvcc_path(), *flags, "-MD", "-MF", obj + ".d", "-c", "-o", obj, src]
        if verbose:
            print(" ".join(cmd))
        running.append((cmd, subprocess.Popen(cmd)))
    failed = [cmd for cmd, p in running if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    subprocess.check_call([nvcc_path(), *ARCH, "--shared", "-cudart", "static", "-Xlinker", "-soname=" + os.path.basename(LIB),
                           "-o", LIB + ".tmp", *objects])
    os.replace(LIB + ".tmp", LIB)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    sys.exit(0)
