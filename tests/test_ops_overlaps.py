"""Buffers of the cache and beam operators that lie on one another are refused, and every refusal names its argument, on the CPU:
each check comes before the GPU is touched (no compute calls here)."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).parent


def _built(src, exe, *more):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    subprocess.run(["g++", "-std=c++17", "-O1", str(HERE / src), "-o", str(exe), *more], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)


def test_sets_of_strided_pieces(mit2, tmp_path):
    run = _built("overlaps.cpp", tmp_path / "overlaps", f"-I{mit2.PKG_DIR / 'csrc'}")
    assert run.returncode == 0, run.stdout + run.stderr


def test_each_refusal_is_for_its_argument(mit2, tmp_path):
    run = _built("ops_messages.cpp", tmp_path / "ops_messages", f"-I{mit2.HEADER_PATH.parent}", str(mit2.LIB_PATH), f"-Wl,-rpath,{mit2.LIB_PATH.parent}",
                 "-Wl,--allow-shlib-undefined")
    assert run.returncode == 0 and ", 0 wrong" in run.stdout, run.stdout + run.stderr
