"""kv8_floor_sum, which the shares of sdv_kv8_plan.h are worked out with, against the sum term by term."""
from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from conftest import ROOT

CSRC = ROOT / "specdec-context-scaling_amd" / "csrc"


def test_floor_sums(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not found")
    exe = tmp_path / "floor_sum_check"
    subprocess.run([cxx, "-O2", "-Wall", "-Werror", f"-I{CSRC}", "-o", str(exe), str(ROOT / "tests" / "native" / "floor_sum_check.cpp")], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    m = re.fullmatch(r"(\d+) sums, (\d+) differences\n", res.stdout)
    assert m and res.returncode == 0, res.stdout + res.stderr
    assert int(m[1]) > 3_000_000 and int(m[2]) == 0
