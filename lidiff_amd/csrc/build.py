"""Builds liblidiff_amd.so (HIP kernels + C ABI) in-tree for gfx950 with hipcc.

    python -m lidiff_amd.csrc.build [--force]

hipcc cross-compiles without a GPU, so this also runs in the CPU-only build container.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCES = ["coords.hip", "spconv.hip", "spconv_rows.hip", "spconv_bf16.hip", "spconv_split3.hip", "norm.hip", "step.hip", "head.hip",
           "groupnorm.hip", "attention_fwd.hip", "attention_bwd.hip"]
# step.hip restates a sequence of separately rounded torch launches: no fused multiply-adds there
EXTRA_FLAGS = {"step.hip": ["-ffp-contract=off"]}
HEADERS = ["common.h", "spconv.h", "segments.h", "attention.h", os.path.join("..", "..", "include", "lidiff_amd.h")]
LIB = os.path.join(HERE, "liblidiff_amd.so")
ARCH = "gfx950"
# no packed fp32 instructions (v_pk_add / mul / fma_f32): every fp32 operation is its own instruction
NO_PACKED_F32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: the lidiff_amd HIP extension cannot be built")


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(HERE, s) for s in SOURCES + HEADERS] + [os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    headers = max(os.path.getmtime(os.path.join(HERE, h)) for h in HEADERS)
    me = os.path.getmtime(os.path.abspath(__file__))

    def compile_one(src: str) -> str:
        path, obj = os.path.join(HERE, src), os.path.join(HERE, src.replace(".hip", ".o"))
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > max(headers, me, os.path.getmtime(path)):
            return obj
        cmd = [_hipcc(), f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-x", "hip",
               "-c", path, "-o", obj] + NO_PACKED_F32 + EXTRA_FLAGS.get(src, [])
        if verbose:
            cmd.insert(1, "-Rpass-analysis=kernel-resource-usage")
        subprocess.run(cmd, check=True)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as pool:          # the sources are independent of each other
        objs = list(pool.map(compile_one, SOURCES))
    subprocess.run([_hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", LIB] + objs, check=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
