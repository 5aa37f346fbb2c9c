"""How the attention weights' launches are laid out (kv_plan.h), on the host: over the sizes that its calls accept, and at the sizes by which
test_gpu_kv_weigh_queries.py means to reach the waves that divide the queries."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

import weigh_cases as cases  # noqa: E402
from ops_ref import Batch  # noqa: E402


@pytest.fixture(scope="module")
def exe(mit2, tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = tmp_path_factory.mktemp("weigh") / "weigh_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{mit2.PKG_DIR / 'csrc'}", str(Path(__file__).parent / "weigh_plan.cpp"), "-o", str(exe)], check=True)
    return exe


def test_plans_can_be_launched(exe):
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and " 0 wrong" in run.stdout, run.stdout + run.stderr


def plans(mit2, exe, batches):
    """(by_query, blocks, by_xcd) of each (batch, last_rows, weight_stride, max_length)."""
    lines = [f"{mit2.DTYPES[b.dtype]} {b.dim} {b.kv_heads} {b.q_heads // b.kv_heads} {len(b.new)} {b.rows} {max(b.length) if hint is None else hint} {b.page} "
             f"{b.table.shape[1]} {last} {stride or b.table.shape[1] * b.page}\n" for b, last, stride, hint in batches]
    run = subprocess.run([str(exe), "-"], input="".join(lines), capture_output=True, text=True, timeout=120, check=True)
    return [tuple(int(x) for x in line.split()) for line in run.stdout.splitlines()]


def test_sizes_reach_the_waves_that_divide_the_queries(mit2, exe):
    listed = [(c, 0, None) for c in cases.SIZES + cases.BIRTHS + cases.XCD + cases.FINITE + cases.QUERIES + [cases.LONG]]
    listed += [(c, 0, stride) for stride, c in cases.STRIDES]
    listed += [(c, cases.LAST if name == "last" else 0, None) for name, c in cases.OTHERS.items()]
    batches = [(Batch(**c["args"]), last, stride, None) for c, last, stride in listed]
    for (c, _, stride), (by_query, blocks, by_xcd) in zip(listed, plans(mit2, exe, batches)):
        assert by_query and bool(by_xcd) == c["by_xcd"], (c, stride, by_query, blocks, by_xcd)
    for hint in (0, 1, 100, 1 << 20, 2 ** 32 - 1):
        assert plans(mit2, exe, [(Batch(**cases.LONG["args"]), 0, None, hint)])[0][0], hint


def test_the_said_length_chooses_the_form(mit2, exe):
    for c in cases.HINTED:
        b = Batch(**c["args"])
        assert all(by_query for by_query, _, _ in plans(mit2, exe, [(b, 0, None, hint) for hint in cases.FEW])), c
        assert not any(by_query for by_query, _, _ in plans(mit2, exe, [(b, 0, None, hint) for hint in cases.MANY])), c
