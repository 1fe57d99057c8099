"""Build libfp4gemm.so in place (sm_100a only).

``python fp4-gemm-blackwell_b200/build.py`` compiles every CUDA source in
``csrc/`` with nvcc for ``sm_100a`` into ``libfp4gemm.so`` beside
``fp4_gemm.py`` (the layout fp4_gemm.py:26-27 of the reference expects).
nvcc cross-compiles without a GPU.  The CUDA runtime is linked statically, so
the library only needs the driver at run time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libfp4gemm.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

SOURCES = ["capi.cu", "quantize.cu", "quantize_units.cu", "gemm_sm100.cu", "noalloc.cu", "selftest.cu", "peak.cu", "peer_barrier.cu",
           "kv_cache.cu", "decode_attention.cu", "gemv.cu"]
HEADERS = ["decode_core.cuh", "fp4b_internal.h", "nvfp4_codec.cuh", "ptx_sm100.cuh", "quantize_core.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
    "-shared",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise FileNotFoundError("nvcc not found")


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in SOURCES + HEADERS] + [os.path.join(INCLUDE, "fp4gemm.h"), __file__]
    return all(os.path.getmtime(d) <= t for d in deps if os.path.exists(d))


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> str:
    if not force and up_to_date():
        return LIB
    # One nvcc per source, as many at a time as there are cores, then the link.
    cc = nvcc()
    tmp = LIB + ".tmp"
    with tempfile.TemporaryDirectory(prefix="fp4b_build_") as work:
        def compile_one(name: str) -> str:
            obj = os.path.join(work, name + ".o")
            cmd = [cc, *[f for f in NVCC_FLAGS if f != "-shared"], *(extra or []), f"-I{CSRC}", f"-I{INCLUDE}",
                   "-c", os.path.join(CSRC, name), "-o", obj]
            if verbose:
                print(" ".join(cmd))
            subprocess.check_call(cmd)
            return obj

        with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
            objs = list(pool.map(compile_one, SOURCES))
        subprocess.check_call([cc, *NVCC_FLAGS, *objs, "-o", tmp])
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    extra = [a for a in sys.argv[1:] if a.startswith("-X") or a.startswith("--")]
    extra = [a for a in extra if a not in ("--force", "--verbose")]
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, extra=extra))
