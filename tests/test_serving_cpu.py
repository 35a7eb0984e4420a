"""Serving operators without a GPU: refusals and error paths of every entry point on a
stand-in HIP runtime (serving_check.c), the paged cache's index arithmetic
(serving_geom_check.cpp), and the MFMA guards of the new kernels."""
import os
import shutil
import subprocess

import pytest

import lpta
from lpta import _native
from test_mfma_exec_cpu import CSRC, _asm, _hipcc, exposed_mfmas

HERE = os.path.dirname(os.path.abspath(__file__))
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(shutil.which("gcc") is None or not os.path.isdir(os.path.join(ROCM, "include", "hip")),
                    reason="gcc or the HIP headers are not available")
def test_refusals_and_error_paths(tmp_path):
    lib = lpta.load_library()._name
    exe = tmp_path / "serving_check"
    subprocess.run(["gcc", "-O1", "-D__HIP_PLATFORM_AMD__", "-rdynamic", "-o", str(exe),
                    os.path.join(HERE, "serving_check.c"), "-I", os.path.join(ROCM, "include"), "-I", INCLUDE, lib,
                    "-Wl,-rpath," + os.path.dirname(lib), "-Wl,-rpath," + os.path.join(ROCM, "lib"),
                    "-Wl,-rpath-link," + os.path.join(ROCM, "lib")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and ", 0 wrong" in out.stdout, out.stdout + out.stderr


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")
def test_paged_index_arithmetic(tmp_path):
    exe = tmp_path / "geom"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", "-o", str(exe),
                    os.path.join(HERE, "serving_geom_check.cpp"), "-I", CSRC], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "0 wrong", out.stdout + out.stderr


def test_paged_cache_layout_matches_header(tmp_path):
    fields = [f for f, _ in _native.TlPagedCache._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "tl_int8.h"\nint main(void) {\n'
                   + "".join(f'    printf("%zu\\n", offsetof(tl_paged_cache, {f}));\n' for f in fields)
                   + '    printf("%zu %d %d %d %d\\n", sizeof(tl_paged_cache), TL_F32, TL_BF16, TL_F16, TL_I8);\n'
                   + "    return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", INCLUDE, "-o", str(exe), str(src)], check=True)
    import ctypes
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(_native.TlPagedCache, f).offset for f in fields] + [
        ctypes.sizeof(_native.TlPagedCache), _native.TL_F32, _native.TL_BF16, _native.TL_F16, _native.TL_I8]


@pytest.mark.skipif(_hipcc() is None, reason="hipcc is needed to compile the kernels")
@pytest.mark.parametrize("src", ["tl_paged.hip", "tl_w4.hip", "tl_score.hip"])
def test_no_mfma_runs_under_a_narrowed_exec(src, tmp_path):
    hits = exposed_mfmas(_asm(os.path.join(CSRC, src), str(tmp_path)))
    assert hits == [], f"MFMAs under a narrowed EXEC with no skip in {src}: {hits[:10]}"
