"""Build the sm_100a shared libraries behind fa2.kernel, fa2.rotary and fa2.kvcache.

    python triton-fa2-forward_b200/build.py          # or: __graft_entry__.build()

Compiles csrc/*.cu with nvcc for sm_100a only (-gencode arch=compute_100a,code=sm_100a)
into fa2/libfa2_sm100.so (attention, include/fa2_sm100.h) and fa2/libfa2_kvcache_sm100.so (rotary
positions and the 8-bit K/V cache, include/fa2_kvcache_sm100.h), in-tree, so they travel with the
source tree. The CUDA runtime is linked statically; the libraries have no torch dependency and
export only the C ABI of their headers.
"""

import os
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_PATH = os.path.join(PKG_DIR, "fa2", "libfa2_sm100.so")
SOURCES = [os.path.join(CSRC, "fa2_fwd_sm100.cu")]
DEPENDS = SOURCES + [
    os.path.join(CSRC, "ptx_sm100.cuh"),
    os.path.join(CSRC, "exp2_poly.cuh"),
    os.path.join(CSRC, "fa2_pair_sm100.cuh"),
    os.path.join(INCLUDE, "fa2_sm100.h"),
]

KV_LIB_PATH = os.path.join(PKG_DIR, "fa2", "libfa2_kvcache_sm100.so")
KV_SOURCES = [os.path.join(CSRC, f) for f in ("rotary_sm100.cu", "kv8_cache_sm100.cu", "kv8_attn_sm100.cu")]
KV_DEPENDS = KV_SOURCES + [os.path.join(CSRC, f) for f in ("kv8_common.cuh", "kv8_attn.cuh", "kv8_chunk.cuh", "ptx_sm100.cuh")] + [
    os.path.join(INCLUDE, "fa2_sm100.h"),
    os.path.join(INCLUDE, "fa2_kvcache_sm100.h"),
]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC,-fvisibility=hidden",
    "-cudart", "static",
]


def nvcc_path():
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def up_to_date(out=LIB_PATH, deps=DEPENDS):
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(d) <= t for d in deps)


def _command(out, sources, extra_flags):
    return [nvcc_path(), *NVCC_FLAGS, *extra_flags, "-I", INCLUDE, "-I", CSRC, "-o", out, *sources]


def build(force=False, verbose=False, extra_flags=()):
    """Compile each library if any of its sources is newer than it (both at the same time). Returns
    the attention library's path."""
    wanted = [(LIB_PATH, SOURCES, DEPENDS, list(extra_flags)), (KV_LIB_PATH, KV_SOURCES, KV_DEPENDS, ["--threads", "0"])]
    running = []
    for out, sources, deps, flags in wanted:
        if force or not up_to_date(out, deps):
            cmd = _command(out, sources, flags)
            if verbose:
                print(" ".join(cmd), flush=True)
            running.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
    said = [(r, *r.communicate()) for r in running]
    for r, out, err in said:
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed ({r.returncode}):\n{out}\n{err}")
        if verbose and (out or err):
            print(out, err, sep="\n")
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
