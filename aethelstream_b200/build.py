"""Build libaeth_galore.so (sm_100a) in-tree with nvcc.

    python aethelstream_b200/build.py [--force] [--verbose]

Run it as a script (or load it by file path): importing the package itself
requires the built library.

The library is three translation units, compiled side by side: csrc/aeth_galore.cu
(the optimizer step), csrc/aeth_train.cu (the training operators around it) and
csrc/aeth_rotary.cu (queries and keys).
It is linked against the static CUDA runtime, so it only needs the driver on the
machine that loads it.  No fast-math: the NF4/INT8 codes and the REF-mode arithmetic must round
exactly like the CPU definition.
"""
from __future__ import annotations

import argparse
import glob
import os
import re
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libaeth_galore.so")
OBJ = os.path.join(HERE, "_obj")  # object files, kept so an unchanged unit is not compiled again
UNITS = ("aeth_galore", "aeth_train", "aeth_rotary")
ROOT = os.path.dirname(HERE)

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2,-ffp-contract=off",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) +
                  [os.path.join(ROOT, "include", "aeth_galore.h")])


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(s) > t for s in sources())


def stale(obj: str, unit: str) -> bool:
    """Whether `unit`'s object is missing or older than the unit or any file it
    includes (found by following the quoted includes)."""
    if not os.path.exists(obj):
        return True
    seen, todo = set(), [os.path.join(CSRC, unit + ".cu")]
    while todo:
        f = os.path.normpath(todo.pop())
        if f in seen:
            continue
        seen.add(f)
        with open(f) as h:
            todo += [os.path.join(os.path.dirname(f), m) for m in re.findall(r'^#include "([^"]+)"', h.read(), re.M)]
    return any(os.path.getmtime(f) > os.path.getmtime(obj) for f in seen)


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> str:
    if not force and not needs_build():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    suffix = ".extra.o" if extra else ".o"  # objects with flags of their own serve this build alone
    objects = [os.path.join(OBJ, unit + suffix) for unit in UNITS]
    compiles = []
    for unit, obj in zip(UNITS, objects):
        src = os.path.join(CSRC, unit + ".cu")
        if force or extra or stale(obj, unit):
            cmd = [nvcc(), *NVCC_FLAGS, *(extra or []), "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj[:-2] + ".part.o"]
            if verbose:
                print(" ".join(cmd))
            compiles.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for obj, p in compiles:
        out = p.communicate()[0]
        if p.returncode != 0:
            sys.stderr.write(out)
        else:
            os.replace(obj[:-2] + ".part.o", obj)  # whole, or not at all
            if verbose and out:
                print(out)
    if any(p.returncode != 0 for _, p in compiles):
        raise RuntimeError("nvcc failed building libaeth_galore.so")
    cmd = [nvcc(), *NVCC_FLAGS[:2], "-shared", *objects, "-o", LIB + ".tmp"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed linking libaeth_galore.so")
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-v", action="store_true", help="print per-kernel register/smem usage")
    a = ap.parse_args()
    build(force=a.force or a.ptxas_v, verbose=a.verbose or a.ptxas_v, extra=["-Xptxas", "-v"] if a.ptxas_v else None)
    print(LIB)
