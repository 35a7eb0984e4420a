"""That the sizes of w8_paths.py take every way through the 8-bit projections' kernels, by their plans."""
import os
import shutil
import subprocess

import pytest

from test_mfma_exec_cpu import CSRC
from w8_paths import PAST_ROWS, ROW_CASES, TILE_CASES, TILED

HERE = os.path.dirname(os.path.abspath(__file__))
ROW, SPLIT, TILE = range(3)
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")


def plans(cases, tmp_path):
    exe = tmp_path / "plans"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-o", str(exe), os.path.join(HERE, "w8_paths_plan.cpp"), "-I", CSRC],
                   check=True)
    asked = "".join(f"{m} {n} {k} {int(g)}\n" for m, n, k, g in cases)
    out = subprocess.run([str(exe)], input=asked, capture_output=True, text=True, check=True).stdout
    got = [tuple(map(int, line.split())) for line in out.splitlines()]
    assert len(got) == len(cases)
    return got


def test_tiled_form(tmp_path):
    """Every shape, alone and gated where it can be, with no pass of the ring's loop and each number of last stages,
    with one and two passes and each number, and with many."""
    seen = set()
    for (m, n, k, gated), (kind, _, _, _, shape, blocks, _) in zip(TILE_CASES, plans(TILE_CASES, tmp_path)):
        assert kind == TILE and TILED[gated][shape] == (m, n), (m, n, k, gated)
        passes, left = 0, blocks
        while left >= 8:
            passes, left = passes + 1, left - 4
        seen.add((gated, shape, min(passes, 3), left))
    ways = {(0, 2), (0, 4), (0, 6), (1, 4), (1, 6), (2, 4), (2, 6), (3, 4)}
    assert seen == {(gated, shape, *w) for gated in TILED for shape in TILED[gated] for w in ways}
    assert set(TILED[False]) == {0, 1, 2, 3}


def test_single_rows(tmp_path):
    """Every number of units of a row that a thread holds with every number of rows that go with it, every number of
    wavefronts to a tile, and loops that fetch weights past the first ones."""
    held, splits, loops = set(), set(), set()
    for (m, n, k, gated), (kind, split, _, _, _, blocks, slots) in zip(ROW_CASES, plans(ROW_CASES, tmp_path)):
        assert kind == ROW, (m, n, k, gated)
        held.add((gated, m, slots))
        splits.add((gated, split))
        ahead = 4 if gated else 8
        loops.add((gated, min(blocks // split // ahead, 3)))
    for gated in (False, True):
        assert {(gated, 1, 1), (gated, 1, 2), (gated, 1, 3), (gated, 1, 4), (gated, 2, 1), (gated, 2, 2), (gated, 3, 1),
                (gated, 4, 1)} <= held
        assert {(gated, s) for s in (1, 2, 4, 8)} <= splits
        assert {(gated, n) for n in (1, 2, 3)} <= loops
    assert all(p[0] == SPLIT for p in plans(PAST_ROWS, tmp_path))
