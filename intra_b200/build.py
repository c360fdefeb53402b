"""Builds libintra_b200.so in-tree with nvcc for sm_100a.

    python -m intra_b200.build            # build if sources are newer than the library
    python -m intra_b200.build --force

The library lands in intra_b200/_lib/ next to the sources, so it is found by `intra_b200._loader`
without an install step.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libintra_b200.so")
SOURCES = [os.path.join(CSRC, f) for f in ("capi.cu", "serving.cu")]
# every header next to the sources counts: an edit to any of them must trigger a rebuild
HEADERS = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))) + [
    os.path.join(PKG_DIR, "..", "include", "intra_b200.h")]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put it on PATH")


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    built = os.path.getmtime(LIB_PATH)
    return all(os.path.getmtime(f) <= built for f in SOURCES + HEADERS + [os.path.abspath(__file__)])


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    flags = [nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC"]
    with tempfile.TemporaryDirectory() as tmp:
        objects = [os.path.join(tmp, os.path.basename(f) + ".o") for f in SOURCES]
        cmds = [flags + ["-c", "-Xptxas", "-v", "-o", obj, src] for src, obj in zip(SOURCES, objects)]
        procs = [subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for cmd in cmds]
        said = [p.communicate()[0] for p in procs]          # the sources compile side by side
        failed = any(p.returncode != 0 for p in procs)
        if not failed:
            link = subprocess.run(flags + ["-shared", "-o", LIB_PATH] + objects, capture_output=True, text=True)
            said.append(link.stdout + link.stderr)
            failed = link.returncode != 0
    if verbose or failed:
        sys.stderr.write("".join(said))
    if failed:
        raise RuntimeError("nvcc failed building libintra_b200.so")
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
