"""Build libintcrush_b200.so in place (nvcc, sm_100a only).

Usage: ``python build.py`` from anywhere.  The library is written next to this
file so that it travels with the source tree; it links the CUDA runtime
statically and does not link libcuda (driver entry points are resolved at run
time), so it loads on hosts without a GPU driver.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libintcrush_b200.so")
# translation unit -> the sources it includes
UNITS = {
    "intcrush_b200.cu": ["ic_common.cuh", "register_split.h", "prep_common.cuh", "prep.cu", "prep_tile.cu", "gemm_tc.cu",
                         "skinny.cu", "weights.cu", "abi.cu"],
    "attention_b200.cu": ["ic_common.cuh", "register_split.h", "qk_norm_rope.cu", "lora_batched.cu", "lora_stream.cu", "lora_feed.h",
                          "cross_attention.cuh", "cross_attention.cu", "cross_attention_tc.cu", "abi_attention.cu"],
    "fp8_b200.cu": ["ic_common.cuh", "register_split.h", "quant_fp8.cu", "gemm_fp8.cu", "group_norm.cu", "abi_fp8.cu"],
}
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
         "-diag-suppress", "20044"]


def _nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def _object(unit: str) -> str:
    return os.path.join(HERE, "_build", unit.replace(".cu", ".o"))


def _stale(target: str, unit: str) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    deps = [os.path.join(CSRC, s) for s in [unit, *UNITS[unit]]]
    deps += [os.path.join(HERE, "..", "include", "intcrush_b200.h"), os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def needs_build() -> bool:
    return any(_stale(LIB, u) for u in UNITS)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the units that changed (side by side) and link the library."""
    if not force and not needs_build():
        return LIB
    os.makedirs(os.path.join(HERE, "_build"), exist_ok=True)
    running = []
    for unit in UNITS:
        obj = _object(unit)
        if not force and not _stale(obj, unit):
            continue
        cmd = [_nvcc(), *FLAGS, "-c", "-o", obj + ".tmp", os.path.join(CSRC, unit)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        running.append((subprocess.Popen(cmd), cmd, obj))
    failed = [(p.returncode, cmd) for p, cmd, _ in running if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(*failed[0])
    for _, _, obj in running:
        os.replace(obj + ".tmp", obj)
    subprocess.run([_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "--shared", "-cudart", "static", "-o",
                    LIB + ".tmp", *map(_object, UNITS)], check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
