"""Which workgroups of the paged attention's joining kernel join what, on the CPU (paged_join_check.cpp)."""
import os
import shutil
import subprocess

import pytest

from test_mfma_exec_cpu import CSRC

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")
def test_every_split_row_is_joined_once(tmp_path):
    exe = tmp_path / "join"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", "-o", str(exe),
                    os.path.join(HERE, "paged_join_check.cpp"), "-I", CSRC], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "0 wrong", out.stdout + out.stderr
