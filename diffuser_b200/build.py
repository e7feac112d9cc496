"""Build the sm_100a engine library (``_lib/libdqlinear.so``) with nvcc.

Every ``csrc/*.cu`` is one translation unit, compiled for ``sm_100a`` only into
``_lib/build/`` (all that are out of date at once: ``dq_capi.cu`` alone takes
minutes) and linked against the static CUDA runtime; the library exports the C
ABI declared in ``include/``.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_DIR = os.path.join(HERE, "_lib")
OBJ_DIR = os.path.join(LIB_DIR, "build")
LIB_PATH = os.path.join(LIB_DIR, "libdqlinear.so")
HEADER = os.path.join(INCLUDE, "dq_linear.h")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [*ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]


def _sources():
    srcs = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC))
            if f.endswith((".cu", ".cuh", ".h"))]
    return srcs + [os.path.join(INCLUDE, f) for f in sorted(os.listdir(INCLUDE)) if f.endswith(".h")]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the sm_100a library cannot be built")
    return cand


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    return all(os.path.getmtime(s) <= t for s in _sources())


def _object_fresh(obj: str) -> bool:
    """Whether an object is newer than every file its dependency list names."""
    dep = obj[:-2] + ".d"
    if not os.path.exists(obj) or not os.path.exists(dep):
        return False
    with open(dep) as f:
        names = f.read().replace("\\\n", " ").split(":", 1)[1].split()
    t = os.path.getmtime(obj)
    return all(os.path.exists(n) and os.path.getmtime(n) <= t for n in names if n.startswith(ROOT))


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile ``csrc/*.cu`` and link ``_lib/libdqlinear.so`` (skipped when fresh)."""
    if not force and up_to_date():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc, objs, jobs = _nvcc(), [], []
    for name in sorted(f for f in os.listdir(CSRC) if f.endswith(".cu")):
        obj = os.path.join(OBJ_DIR, name[:-3] + ".o")
        objs.append(obj)
        if not force and _object_fresh(obj):
            continue
        cmd = [nvcc, *NVCC_FLAGS, "-MD", "-MF", obj[:-2] + ".d", "-c", "-o", obj + ".tmp",
               os.path.join(CSRC, name)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), file=sys.stderr)
        jobs.append((obj, cmd, subprocess.Popen(cmd)))
    failed = [cmd for _, cmd, p in jobs if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    for obj, _, _ in jobs:
        os.replace(obj + ".tmp", obj)
    tmp = LIB_PATH + ".tmp"
    subprocess.run([nvcc, *ARCH_FLAGS, "-shared", "-o", tmp, *objs], check=True)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
