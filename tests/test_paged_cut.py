"""The varlen attention's cut of its work and its page-list arithmetic (csrc/tsfa_paged.h), built for the host with
-fsanitize=address,undefined: tests/sanitize/paged_cut.cpp."""

import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "eagle3-tree-sparse-flashattn_amd" / "csrc"
GXX = shutil.which("g++")


@pytest.mark.skipif(GXX is None, reason="needs g++")
def test_every_step_belongs_to_one_run(tmp_path):
    exe = tmp_path / "paged_cut"
    subprocess.run([GXX, "-std=c++17", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-g", "-O1",
                    f"-I{CSRC}", str(ROOT / "tests" / "sanitize" / "paged_cut.cpp"),
                    str(CSRC / "tsfa_plan.cpp"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "ASAN_OPTIONS": "detect_leaks=1", "UBSAN_OPTIONS": "print_stacktrace=1"})
    out = res.stdout + res.stderr
    assert res.returncode == 0 and "all invariants hold" in res.stdout, out[-4000:]
