"""Builds libqm38.so (HIP kernels + C-ABI runtime) for gfx950 with hipcc.

Usage: python qwen38-metal_amd/build.py [--jobs N]

Objects go to qwen38-metal_amd/_build/, the library to
qwen38-metal_amd/qm38/libqm38.so (in-tree, so it travels with the source tree).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "qm38" / "libqm38.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

COMMON = [
    "--offload-arch=gfx950",
    "-O3",
    "-fPIC",
    "-std=c++17",
    "-Wall",
    "-Wno-unused-function",
    "-Wno-unused-variable",
    # Packed fp32 VALU ops stay disabled: some of their forms have given
    # wrong results on this hardware; hipcc emits plain fp32 ops instead.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{PKG.parent / 'include'}",
]


# Per-file flags.  Attention: MFMA accumulators in VGPRs (the compiler would
# otherwise park them in AGPRs and copy them back every step).
PER_FILE = {
    "q8_attention.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "q4kv_attention.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    # The score products in VGPRs; the sums then take the AGPRs without copies.
    "latent_expanded.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    "latent_absorbed.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
}


def _compile(src: Path) -> Path:
    obj = BUILD / (src.name + ".o")
    cmd = [HIPCC, *COMMON, *PER_FILE.get(src.name, []), "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    return obj


def build(jobs: int = 8) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip")) + sorted(CSRC.glob("*.cpp"))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, sources))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=8)
    a = ap.parse_args()
    print(build(a.jobs))
    sys.exit(0)
