"""The 8-bit projections, the append with norms and the attention over a shared prefix without a GPU: refusals and
error paths on a stand-in HIP runtime (serving_more_check.c), plans and sizes (w8_plan_check.cpp), and the MFMA guards
of the new kernels."""
import os
import shutil
import subprocess

import pytest

import lpta
from test_mfma_exec_cpu import CSRC, _asm, _hipcc, exposed_mfmas

HERE = os.path.dirname(os.path.abspath(__file__))
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(shutil.which("gcc") is None or not os.path.isdir(os.path.join(ROCM, "include", "hip")),
                    reason="gcc or the HIP headers are not available")
def test_refusals_and_error_paths(tmp_path):
    lib = lpta.load_library()._name
    exe = tmp_path / "serving_more_check"
    subprocess.run(["gcc", "-O1", "-D__HIP_PLATFORM_AMD__", "-rdynamic", "-o", str(exe),
                    os.path.join(HERE, "serving_more_check.c"), "-I", os.path.join(ROCM, "include"), "-I", INCLUDE, lib,
                    "-Wl,-rpath," + os.path.dirname(lib), "-Wl,-rpath," + os.path.join(ROCM, "lib"),
                    "-Wl,-rpath-link," + os.path.join(ROCM, "lib")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and ", 0 wrong" in out.stdout, out.stdout + out.stderr


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")
def test_plans(tmp_path):
    exe = tmp_path / "w8_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", "-o", str(exe),
                    os.path.join(HERE, "w8_plan_check.cpp"), "-I", CSRC], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "0 wrong", out.stdout + out.stderr


@pytest.mark.skipif(_hipcc() is None, reason="hipcc is needed to compile the kernels")
@pytest.mark.parametrize("src", ["tl_prefix.hip", "tl_w8.hip"])
def test_no_mfma_runs_under_a_narrowed_exec(src, tmp_path):
    hits = exposed_mfmas(_asm(os.path.join(CSRC, src), str(tmp_path)))
    assert hits == [], f"MFMAs under a narrowed EXEC with no skip in {src}: {hits[:10]}"
