"""Build libatlas_mem.so in-tree with nvcc for sm_100a (no torch headers needed).

Every csrc/*.cu is one translation unit: the stale ones compile in parallel into _build/*.o,
then all link into one shared library.

    python -m atlas_rnn_b200.build
"""
from __future__ import annotations

import glob
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OBJ_DIR = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "libatlas_mem.so")


def sources() -> list:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def deps(src: str) -> set:
    """A source file and the project headers it includes, directly or not."""
    seen, todo = set(), [src]
    while todo:
        path = todo.pop()
        if path in seen:
            continue
        seen.add(path)
        for name in re.findall(r'^\s*#include "([^"]+)"', open(path).read(), re.M):
            for d in (CSRC, INCLUDE):
                if os.path.exists(os.path.join(d, name)):
                    todo.append(os.path.join(d, name))
    return seen


def obj_of(src: str) -> str:
    return os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")


def _newer(path: str, than: set) -> bool:
    return os.path.exists(path) and all(os.path.getmtime(d) <= os.path.getmtime(path) for d in than)


def nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def up_to_date() -> bool:
    return all(_newer(OUT, deps(s)) for s in sources())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return OUT
    os.makedirs(OBJ_DIR, exist_ok=True)
    arch = ["-gencode", "arch=compute_100a,code=sm_100a"]
    running = []
    for src in sources():
        if not force and _newer(obj_of(src), deps(src)):
            continue
        cmd = [nvcc(), *arch, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I" + INCLUDE, "-c", "-o",
               obj_of(src) + ".tmp", src]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd))
        running.append((subprocess.Popen(cmd), cmd, obj_of(src)))
    failed = [(p.wait(), cmd) for p, cmd, _ in running]
    for rc, cmd in failed:
        if rc:
            raise subprocess.CalledProcessError(rc, cmd)
    for _, _, obj in running:
        os.replace(obj + ".tmp", obj)
    subprocess.run([nvcc(), *arch, "-shared", "-o", OUT + ".tmp"] + [obj_of(s) for s in sources()], check=True)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
