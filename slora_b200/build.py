"""Build ``libslora_b200.so`` in-tree with nvcc for sm_100a:  ``python slora_b200/build.py [--force] [-v]``.

Run as a script (or load this file by path): importing the package needs the library to exist already.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SOURCES = [os.path.join(HERE, "csrc", f) for f in ("lora_kernels.cu", "kv_kernels.cu")]
HEADERS = [os.path.join(ROOT, "include", "slora_b200.h")] + sorted(
    os.path.join(HERE, "csrc", f) for f in os.listdir(os.path.join(HERE, "csrc")) if f.endswith((".cuh", ".h")))
OBJECTS = os.path.join(HERE, "build")
OUT = os.path.join(HERE, "libslora_b200.so")

NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
              "-I", os.path.join(ROOT, "include")]


def _stale(target, sources):
    return not os.path.exists(target) or any(os.path.getmtime(p) > os.path.getmtime(target) for p in sources)


def _headers_of(source, seen=None):
    """The project headers a source file includes, directly or not (by their names in ``HEADERS``)."""
    seen = set() if seen is None else seen
    with open(source) as f:
        lines = [x.split('"')[1] for x in f if x.startswith('#include "')]
    for name in lines:
        for h in HEADERS:
            if os.path.basename(h) == name and h not in seen:
                seen.add(h)
                _headers_of(h, seen)
    return seen


def needs_build():
    return _stale(OUT, SOURCES + HEADERS)


def _run(cmds, verbose):
    procs = [(c, subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)) for c in cmds]
    bad = []
    for cmd, p in procs:
        text = p.communicate()[0]
        if verbose or p.returncode != 0:
            sys.stderr.write(text)
        if p.returncode != 0:
            bad.append(" ".join(cmd))
    if bad:
        raise RuntimeError("nvcc failed: " + "; ".join(bad))


def build(force=False, verbose=False):
    """Compile the CUDA sources, side by side, and link them into ``libslora_b200.so`` (what is up to date is skipped
    unless ``force``)."""
    if not force and not needs_build():
        return OUT
    nvcc = os.environ.get("NVCC", "nvcc")
    os.makedirs(OBJECTS, exist_ok=True)
    objects = [os.path.join(OBJECTS, os.path.basename(p)[:-3] + ".o") for p in SOURCES]
    flags = NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else [])
    _run([[nvcc] + flags + ["-c", src, "-o", obj] for src, obj in zip(SOURCES, objects)
          if force or _stale(obj, [src] + sorted(_headers_of(src)))], verbose)
    _run([[nvcc] + NVCC_FLAGS + ["-shared"] + objects + ["-o", OUT]], verbose)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
