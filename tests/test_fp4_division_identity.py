"""The 4-bit quantizer divides by block scales, and by six, with Newton's iteration and Markstein's correction step;
tests/native/fp4_division_check.c compares them with C's IEEE division for every significand."""

import shutil
import subprocess
from pathlib import Path

import pytest

SRC = Path(__file__).resolve().parent / "native" / "fp4_division_check.c"


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_steps_equal_ieee_division(tmp_path):
    exe = tmp_path / "fp4_division_check"
    subprocess.run(["gcc", "-O2", "-ffp-contract=off", "-fno-fast-math", "-o", str(exe), str(SRC), "-lm"], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    counts = [tuple(int(v) for v in line.split()) for line in res.stdout.splitlines()]
    assert counts == [(8 * 5, 0), (8 * 2 * (1 << 23), 0), (1 << 23, 0)]
    assert res.returncode == 0
