"""CPU test of the prompts' launch shapes: tests/native/prefill_plan.cpp, built against
the library and run."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HIPCC = Path("/opt/rocm/bin/hipcc")


def test_prefill_plans(tmp_path):
    if not HIPCC.exists():
        pytest.skip("hipcc is not installed")
    lib = ROOT / "qwen38-metal_amd" / "qm38"
    exe = tmp_path / "prefill_plan"
    subprocess.run([str(HIPCC), "--offload-arch=gfx950", "-O1", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", f"-I{ROOT / 'include'}", str(ROOT / "tests" / "native" / "prefill_plan.cpp"),
                    f"-L{lib}", "-lqm38", f"-Wl,-rpath,{lib}", "-o", str(exe)], check=True, capture_output=True,
                   text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
