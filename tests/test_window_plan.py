"""How hkv_window_attn cuts its tiles (hkv_plan.h), on the CPU: the parts fit the workspace that an engine
takes when it is made."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


def test_parts_fit_the_workspace(tmp_path):
    gxx = shutil.which("g++", path="/usr/bin:/bin")
    cuda = Path("/usr/local/cuda/include")
    if gxx is None or not (cuda / "cuda_runtime.h").exists():
        pytest.skip("no system g++ or CUDA headers")
    exe = tmp_path / "window_plan_test"
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{REPO / 'higgs-audio.cpp_b200' / 'csrc'}",
                    f"-I{cuda}", str(REPO / "tests" / "cpp" / "window_plan_test.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "window plan ok" in res.stdout
