"""Build the CUDA extension in-tree: kfold_b200/_C/libkfold_b200.so (sm_100a only).

    python -m kfold_b200.build [--verbose] [--force]

Each .cu file is compiled to an object with nvcc (in parallel) and linked into one
shared library that exports the C ABI declared in include/kfold_b200.h.  Objects are
rebuilt only when a source, a header or this file, which has their flags, is newer.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OUT_DIR = os.path.join(PKG, "_C")
LIB = os.path.join(OUT_DIR, "libkfold_b200.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--use_fast_math", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr", "-rdc=true",
]
# Where gates of float32 logits are to be those of elementary float32 operations: what --use_fast_math says but for the fast exponential.
EXACT_EXP = {"residual_norm.cu", "residual_norm_grad.cu"}
EXACT_EXP_FLAGS = ["-ftz=true", "-prec-div=false", "-prec-sqrt=false"]


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _shared_mtime() -> float:
    """Of what every object hangs on."""
    shared = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    shared += [os.path.join(os.path.dirname(PKG), "include", "kfold_b200.h"), os.path.abspath(__file__)]
    return max(os.path.getmtime(f) for f in shared)


def build(verbose: bool = False, force: bool = False) -> str:
    os.makedirs(OUT_DIR, exist_ok=True)
    shared_m = _shared_mtime()
    jobs, objs = [], []
    for src in _sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(OUT_DIR, src[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), shared_m):
            flags = [f for f in FLAGS if f != "--use_fast_math"] + EXACT_EXP_FLAGS if src in EXACT_EXP else FLAGS
            cmd = [NVCC, *flags, "-c", s, "-o", o]
            if verbose:
                cmd.insert(1, "-Xptxas")
                cmd.insert(2, "-v")
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for cmd, r in ex.map(run, jobs):
                if verbose or r.returncode != 0:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed on {cmd[-3]}")
    if jobs or not os.path.exists(LIB):
        cmd = [NVCC, "-shared", "-o", LIB, *objs, "-Xcompiler", "-fvisibility=hidden", "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return LIB


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv, force="--force" in sys.argv))
