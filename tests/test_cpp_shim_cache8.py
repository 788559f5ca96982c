"""The C++ pipeline shim's 8-bit runtime and window_layer: refusals on a host-only engine, and on
the GPU a prompt's rows at once against the same rows one step at a time."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


def build(tmp_path):
    gxx = shutil.which("g++", path="/usr/bin:/bin")
    cuda = Path("/usr/local/cuda")
    if gxx is None or not (cuda / "include" / "cuda_runtime.h").exists():
        pytest.skip("no system g++ or CUDA headers")
    lib_dir = REPO / "higgs-audio.cpp_b200" / "lib"
    exe = tmp_path / "shim_cache8_test"
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{REPO / 'include'}", f"-I{cuda / 'include'}",
                    str(REPO / "tests" / "cpp" / "shim_cache8_test.cpp"), f"-L{lib_dir}", "-lhkv",
                    f"-L{cuda / 'lib64'}", "-lcudart", f"-Wl,-rpath,{lib_dir}:{cuda / 'lib64'}", "-o", str(exe)],
                   check=True)
    return str(exe)


def run(*args):
    res = subprocess.run(args, capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "shim cache8 ok" in res.stdout


def test_cache_type_and_refusals(hkv_lib, tmp_path):
    run(build(tmp_path))


@pytest.mark.gpu
def test_window_layer_is_the_steps(hkv_lib, tmp_path):
    run(build(tmp_path), "gpu")
