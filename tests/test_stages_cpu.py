"""The matrix tiles' copies and waits, replayed on the CPU for every tile that the
sources name: tests/native/stages_check.cpp over csrc/stages.hpp."""
import glob
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "welvet.metal_amd", "csrc")
SRC = os.path.join(ROOT, "tests", "native", "stages_check.cpp")
OUT = os.path.join(ROOT, "welvet.metal_amd", "_build", "stages")


def tiles():
    """(parts, WM, WN, TM, TN, SA, SB) of every Tile<> in the sources; kParts is
    rows8_backward.hip's number of parts."""
    found = set()
    for path in glob.glob(os.path.join(CSRC, "*.hip")):
        with open(path) as f:
            for args in re.findall(r"= Tile<\w+, ([^>]*)>", f.read()):
                parts, *rest = [a.strip() for a in args.split(",")]
                rest = [int(r) for r in rest] + [3, 2][len(rest) - 4:]
                found.add((2 if parts == "kParts" else int(parts), *rest))
    return sorted(found)


@pytest.fixture(scope="module")
def check():
    exe = os.path.join(OUT, "stages_check")
    os.makedirs(OUT, exist_ok=True)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, SRC, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return exe


def test_the_sources_tiles_are_found():
    """Five of one part in int8.hip, four of two in rows8_backward.hip."""
    assert len(tiles()) == 9 and (2, 2, 4, 1, 1, 6, 6) in tiles()


@pytest.mark.parametrize("parts,wm,wn,tm,tn,sa,sb", tiles())
def test_copies_end_before_they_are_read(check, parts, wm, wn, tm, tn, sa, sb):
    waves = wm * wn
    loads = [wm * tm * 32 // 8 // waves, wn * tn * 32 // 8 // waves]
    r = subprocess.run([check, *map(str, (parts, sa, sb, *loads, 300))], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "stages_check: ok" in r.stdout, r.stdout[-2000:]
