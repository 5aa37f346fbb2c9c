"""How the paged attention's launches are laid out (kv_plan.h), on the host over the sizes that its calls accept."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest


def test_plans_can_be_launched_and_cover_the_keys(mit2, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "attend_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{mit2.PKG_DIR / 'csrc'}", str(Path(__file__).parent / "attend_plan.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and " 0 wrong" in run.stdout, run.stdout + run.stderr
