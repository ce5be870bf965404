"""Builds libt2sc.so in-tree (next to this file, under t2sc/) with nvcc for sm_100a.

Usage: python build.py [--force]. Called by __graft_entry__.build().
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
OUT = os.path.join(HERE, "t2sc", "libt2sc.so")
SOURCES = ["api.cu", "hashmap.cu", "scan.cu", "conv_tc.cu", "conv_simt.cu", "convert.cu", "subdiv.cu", "selftest.cu", "norm.cu", "dist.cu", "block.cu", "pipeline.cu", "dense.cu", "dense_tc.cu", "dense_rows.cu", "dense_skinny.cu",
           "rope.cu", "attention.cu", "attention_tc.cu", "attention_rows.cu", "synth.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _stale():
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(HERE, "..", "include", "t2sc.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False):
    if not force and not _stale():
        return OUT
    nvcc = os.environ.get("NVCC", "nvcc")
    flags = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr"]
    if verbose:
        flags += ["-Xptxas", "-v"]
    os.makedirs(OBJ, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers += [os.path.join(HERE, "..", "include", "t2sc.h"), os.path.abspath(__file__)]
    newest = max(os.path.getmtime(h) for h in headers)

    def one(src):  # an object per source, kept while it is newer than the source and every header
        path, obj = os.path.join(CSRC, src), os.path.join(OBJ, src + ".o")
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(newest, os.path.getmtime(path)):
            subprocess.run([nvcc, *flags, "-c", path, "-o", obj + ".tmp"], check=True)
            os.replace(obj + ".tmp", obj)
        return obj

    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        objects = list(pool.map(one, SOURCES))
    subprocess.run([nvcc, *ARCH, "-shared", "-o", OUT + ".tmp", *objects, "-lpthread", "-ldl"], check=True)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
