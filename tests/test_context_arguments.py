"""What the operators for long and shared contexts refuse, and their argument structures and workspaces, on the CPU: every check
comes before the GPU is touched (no compute calls here)."""
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
    exe = tmp_path_factory.mktemp("context") / "context_refusals"
    src = Path(__file__).parent / "context_refusals.cpp"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{mit2.HEADER_PATH.parent}", str(src), str(mit2.LIB_PATH), "-o", str(exe),
                    f"-Wl,-rpath,{mit2.LIB_PATH.parent}", "-Wl,--allow-shlib-undefined"], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)


def test_each_refusal_is_for_its_argument(refusals):
    assert refusals.returncode == 0 and ", 0 wrong" in refusals.stdout, refusals.stdout + refusals.stderr


def test_the_binding_has_the_header_s_structures(mit2, refusals):
    names, last = ("KvNorm", "KvPrefix", "KvWeigh", "KvEvict"), ("eps", "lse", "born", "workspace_bytes")
    lines = {x.split()[0]: [int(v) for v in x.split()[1:]] for x in refusals.stdout.splitlines() if x.startswith(("sizes", "offsets"))}
    assert [ctypes.sizeof(getattr(mit2, n)) for n in names] == lines["sizes"]
    assert [getattr(getattr(mit2, n), f).offset for n, f in zip(names, last)] == lines["offsets"]


def test_null_contexts_and_structures(mit2):
    L = mit2.lib()
    c, r = mit2.KvCache(), mit2.KvRows()
    assert L.mit2cfm_kv_norm_append_device(None, c, r, mit2.KvAppend(), mit2.KvNorm(), 0) == mit2.E_ARG
    assert b"ctx" in L.mit2cfm_last_error(None)
    assert L.mit2cfm_kv_prefix_attention_device(None, c, r, mit2.KvAttention(), mit2.KvPrefix(), 0) == mit2.E_ARG
    assert L.mit2cfm_kv_weigh_device(None, c, r, mit2.KvWeigh(), 0) == mit2.E_ARG
    assert L.mit2cfm_kv_evict_device(None, c, mit2.KvEvict(), 0) == mit2.E_ARG
    assert L.mit2cfm_kv_prefix_attention_workspace(None, None, 1, None) == 0 and L.mit2cfm_kv_evict_workspace(None, None) == 0
    assert mit2.kv_prefix_attention_workspace(c, r, 4, mit2.KvPrefix()) == 0 and mit2.kv_evict_workspace(c, mit2.KvEvict()) == 0


def test_workspaces_follow_their_sizes(mit2):
    c = mit2.KvCache(pages=9, page_rows=16, kv_heads=2, head_dim=64, table_stride=64, dtype=mit2.DTYPE_F16)
    r = mit2.KvRows(start=64, length=64, seqs=4, rows=4, max_length=1000)  # (addresses that nobody reads)
    alone = mit2.kv_prefix_attention_workspace(c, r, 4, mit2.KvPrefix())
    assert 0 < alone < mit2.kv_prefix_attention_workspace(c, r, 4, mit2.KvPrefix(groups=1, max_shared=900))
    assert mit2.kv_prefix_attention_workspace(c, r, 5, mit2.KvPrefix()) == 0  # not a multiple of the key heads
    assert mit2.kv_prefix_attention_workspace(c, r, 4, mit2.KvPrefix(groups=65536)) == 0
    e = mit2.KvEvict(seqs=3, layers=2, weight_stride=1024)
    small = mit2.kv_evict_workspace(c, e)
    # lists of the places that rows leave and come from: half the places each
    assert small >= 3 * 2 * 2 * 1024 * 4
    e.layers = 4
    assert mit2.kv_evict_workspace(c, e) > small
    e.weight_stride = 0
    assert mit2.kv_evict_workspace(c, e) == 0
