"""Build libfta_gfx950.so (hand-written HIP kernels for gfx950 + the C ABI).

Usage: ``python build_lib.py`` (from anywhere).  Objects go to ``_build/``
next to this file; the shared library is written into the Python package
directory so that it travels with the source tree.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
PKG = os.path.join(HERE, "flash_topk_attn_v2")
LIB = os.path.join(PKG, "libfta_gfx950.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

SOURCES = ["fta_api.cpp", "fta_score.hip", "fta_index.hip", "fta_attn.hip", "fta_prep.hip", "fta_window.hip", "fta_cache.hip"]

# Packed fp32 VALU ops are disabled: hipcc -O3 would otherwise form
# v_pk_{add,mul,fma}_f32 from ordinary float code.
COMMON = [
    "-O3",
    "-std=c++17",
    "-fPIC",
    f"--offload-arch={ARCH}",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I", CSRC,
    "-I", os.path.join(os.path.dirname(HERE), "include"),
]

# Matrix instructions that take their operands from VGPRs where the register
# allocator would choose AGPRs: at D = 256 the window backward's dK / dV kernel
# loses all but 75 of its 1312 register copies (120 -> 100 us, 526 -> 422 us over two
# shapes), its dQ kernel pays 6 % (57 -> 60 us, 216 -> 229 us); D <= 128 is unchanged.
EXTRA = {
    "fta_window.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=true"],
}


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.splitext(src)[0] + ".o")
    flags = [*COMMON, *EXTRA.get(src, [])]
    cmd = [HIPCC, *flags, "-c", os.path.join(CSRC, src), "-o", obj]
    if src.endswith(".cpp"):
        cmd = [HIPCC, *flags, "-x", "hip", "-c", os.path.join(CSRC, src), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    return obj


def build(verbose: bool = True) -> str:
    os.makedirs(BUILD, exist_ok=True)
    jobs = min(len(SOURCES), os.cpu_count() or 1, 8)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "-shared", "-fPIC", f"--offload-arch={ARCH}", *objs, "-o", tmp]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build()
    sys.exit(0)
