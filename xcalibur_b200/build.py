"""Build the C-ABI shared library ``libxcb_moe.so`` in-tree with nvcc for sm_100a.

The library has no torch dependency: its entry points take raw device pointers, sizes and a cudaStream_t
(include/xcb_moe.h).  Objects go to ``xcalibur_b200/_build/``; the library lands next to this file so that it
travels with the source tree.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libxcb_moe.so")
SOURCES = ["api.cu", "route.cu", "skinny.cu", "wide.cu", "pack.cu", "probe.cu", "ep.cu", "rope.cu", "attn.cu",
           "pages.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def _flags():
    return ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", os.path.join(ROOT, "include"),
                   "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [
        os.path.join(ROOT, "include", f) for f in ("xcb_moe.h", "xcb_attn.h")]
    return any(os.path.getmtime(d) > t for d in deps)


# Kernels of attn.cu whose warps hand registers to one another start with 128 a thread (launch bounds of two blocks of 256
# threads); with fewer, the ones that take would wait for good, and the library refuses such calls.
_SPLIT = re.compile(r"entry function '\S*attn_kernelI\S*Lb1ELi(?:64|128)ELi[12]E\S*' for.*?Used (\d+) registers", re.S)
_SPLIT_KERNELS = 8


def check_register_split(ptxas: str) -> None:
    """Raise if the compiler's report (``-Xptxas -v``) gives one of these kernels other registers than it hands out."""
    used = [int(n) for n in _SPLIT.findall(ptxas)]
    if len(used) != _SPLIT_KERNELS or any((n + 7) // 8 * 8 != 128 for n in used):
        raise RuntimeError(f"attn.cu: its {_SPLIT_KERNELS} kernels with a register split need 128 registers a thread, "
                           f"the compiler gave {used}")


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    os.makedirs(BUILD, exist_ok=True)

    def compile_one(src: str) -> str:
        obj = os.path.join(BUILD, src.replace(".cu", ".o"))
        cmd = [nvcc(), *_flags(), "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        split = src == "attn.cu"
        done = subprocess.run(cmd + (["-Xptxas", "-v"] if split else []), stderr=subprocess.PIPE if split else None, text=True)
        if split:
            sys.stderr.writelines(line for line in done.stderr.splitlines(True)  # the report stays out, if all is well
                                  if done.returncode or not line.startswith(("ptxas info", "    ")))
        done.check_returncode()
        if split:
            check_register_split(done.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        objs = list(pool.map(compile_one, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", tmp, "-lcudart"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
