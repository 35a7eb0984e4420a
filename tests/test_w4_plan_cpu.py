"""Plan, scratch size and addresses of the 4-bit projections on the CPU (w4_plan_check.cpp)."""
import os
import shutil
import subprocess

import pytest

from test_mfma_exec_cpu import CSRC

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")
def test_digits_that_are_read_lie_in_scratch(tmp_path):
    exe = tmp_path / "w4_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", "-o", str(exe),
                    os.path.join(HERE, "w4_plan_check.cpp"), "-I", CSRC], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "0 wrong", out.stdout + out.stderr
