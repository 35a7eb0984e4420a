"""Errors of calls on several threads, on a stand-in HIP runtime (serving_threads_check.c)."""
import os
import shutil
import subprocess

import pytest

import lpta
from test_serving_cpu import HERE, INCLUDE, ROCM


@pytest.mark.skipif(shutil.which("gcc") is None or not os.path.isdir(os.path.join(ROCM, "include", "hip")),
                    reason="gcc or the HIP headers are not available")
def test_errors_on_several_threads(tmp_path):
    lib = lpta.load_library()._name
    exe = tmp_path / "threads"
    subprocess.run(["gcc", "-O1", "-D__HIP_PLATFORM_AMD__", "-rdynamic", "-o", str(exe),
                    os.path.join(HERE, "serving_threads_check.c"), "-I", os.path.join(ROCM, "include"), "-I", INCLUDE, lib,
                    "-lpthread", "-Wl,-rpath," + os.path.dirname(lib), "-Wl,-rpath," + os.path.join(ROCM, "lib"),
                    "-Wl,-rpath-link," + os.path.join(ROCM, "lib")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "0 wrong", out.stdout + out.stderr
