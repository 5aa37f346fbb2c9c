"""What the cache and beam operators refuse, and their argument structures, on the CPU: every check comes before the GPU is
touched (no compute calls here)."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest


@pytest.fixture(scope="module")
def refusals(mit2, tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = tmp_path_factory.mktemp("ops") / "ops_refusals"
    src = Path(__file__).parent / "ops_refusals.cpp"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{mit2.HEADER_PATH.parent}", str(src), str(mit2.LIB_PATH), "-o", str(exe),
                    f"-Wl,-rpath,{mit2.LIB_PATH.parent}", "-Wl,--allow-shlib-undefined"], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)


def test_bad_arguments_are_refused(refusals):
    assert refusals.returncode == 0, refusals.stdout + refusals.stderr
    assert "0 not refused" in refusals.stdout


def test_the_binding_has_the_header_s_structures(mit2, refusals):
    names = ("KvCache", "KvRows", "KvAppend", "KvAttention", "BeamSelect", "BeamReorder")
    last = ("dtype", "max_length", "theta", "workspace_bytes", "workspace_bytes", "place")
    lines = {x.split()[0]: [int(v) for v in x.split()[1:]] for x in refusals.stdout.splitlines() if x.startswith(("sizes", "offsets"))}
    assert [ctypes.sizeof(getattr(mit2, n)) for n in names] == lines["sizes"]
    assert [getattr(getattr(mit2, n), f).offset for n, f in zip(names, last)] == lines["offsets"]


def test_null_contexts_and_structures(mit2):
    L = mit2.lib()
    c, r, s, o = mit2.KvCache(), mit2.KvRows(), mit2.BeamSelect(), mit2.BeamReorder()
    assert L.mit2cfm_kv_append_device(None, c, r, mit2.KvAppend(), 0) == mit2.E_ARG
    assert b"ctx" in L.mit2cfm_last_error(None)
    assert L.mit2cfm_kv_attention_device(None, c, r, mit2.KvAttention(), 0) == mit2.E_ARG
    assert L.mit2cfm_beam_select_device(None, s, 0) == mit2.E_ARG
    assert L.mit2cfm_beam_reorder_device(None, c, o, 0) == mit2.E_ARG
    assert L.mit2cfm_kv_attention_workspace(None, None, 1) == 0
    assert L.mit2cfm_beam_select_workspace(None) == 0
    assert mit2.kv_attention_workspace(c, r, 4) == 0 and mit2.beam_select_workspace(s) == 0


def test_a_workspace_that_covers_the_sizes(mit2):
    s = mit2.BeamSelect(groups=2, beams=3, vocab=8194, count=6, dtype=mit2.DTYPE_F32, stop_token=-1)
    small = mit2.beam_select_workspace(s)
    s.groups = 4
    assert 0 < small < mit2.beam_select_workspace(s)


def test_pages_and_places(mit2, tmp_path):
    """kv_view.h's arithmetic compiled for the host alone."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not available")
    exe = tmp_path / "kv_pages"
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-std=c++17", "-O1", f"-I{mit2.PKG_DIR / 'csrc'}",
                    str(Path(__file__).parent / "kv_pages.cpp"), "-o", str(exe)], check=True, capture_output=True, timeout=110)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "0 wrong" in run.stdout, run.stdout + run.stderr
