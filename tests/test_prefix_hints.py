"""The shared-prefix attention's plans (kv_plan.h) where the rows are said to be as long as can be, on the host."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest


def test_the_largest_hints_are_the_table_s_length(mit2, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "prefix_hints"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{mit2.PKG_DIR / 'csrc'}", str(Path(__file__).parent / "prefix_hints.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and " 0 wrong" in run.stdout, run.stdout + run.stderr
