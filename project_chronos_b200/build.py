"""Build the sm_100a extension in-tree: project_chronos_b200/libchronos_moe.so.

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

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB = os.path.join(PKG, "libchronos_moe.so")
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


def _up_to_date(obj: str) -> bool:
    """Whether the object is newer than every file nvcc read for it (its .d list)."""
    if not (os.path.exists(obj) and os.path.exists(obj + ".d")):
        return False
    with open(obj + ".d") as f:
        deps = f.read().replace("\\\n", " ").split(":", 1)[1].split()
    t = os.path.getmtime(obj)
    return all(os.path.exists(d) and os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
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
    subprocess.check_call([nvcc_path(), *ARCH, "--shared", "-cudart", "static", "-o", LIB + ".tmp", *objects])
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    sys.exit(0)
