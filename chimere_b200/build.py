"""Build the CUDA library in-tree for sm_100a: chimere_b200/libchimere_b200_moe.so.

    python -m chimere_b200.build            # rebuild if sources are newer than the library
    python -m chimere_b200.build --force

nvcc cross-compiles without a GPU.  The flags are the ones the reference's build scripts use
(chimere-server/ffi/build.rs:103-160: -O3 -std=c++17 -fPIC) with the architecture replaced by
-gencode arch=compute_100a,code=sm_100a.
"""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libchimere_b200_moe.so")
SOURCES = ["abi.cu", "balance.cu", "gemm_i8.cu", "gemv.cu", "gemv_tiled.cu", "gguf.cpp", "kquant.cu", "mma_tiles.cu", "pack.cu", "pairs.cu", "router.cu", "w8a8.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "--compiler-options", "-fPIC", "-shared"]


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "chimere_b200_moe.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    nvcc = os.environ.get("NVCC", "nvcc")

    def run(args: list) -> None:
        r = subprocess.run([nvcc, *args], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
        if verbose:
            print(r.stderr)

    with tempfile.TemporaryDirectory() as objects:      # the sources side by side, the longest take a minute or two each
        compile_flags = [f for f in NVCC_FLAGS if f != "-shared"] + (["-Xptxas", "-v"] if verbose else [])
        paths = [os.path.join(objects, s + ".o") for s in SOURCES]
        with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
            list(pool.map(lambda s, o: run([*compile_flags, "-c", "-o", o, os.path.join(CSRC, s)]), SOURCES, paths))
        run([*NVCC_FLAGS, "-o", LIB, *paths])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
