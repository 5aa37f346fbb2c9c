"""Shared-prefix attention (mit2cfm_kv_prefix_attention_device) of groups whose first sequences have no new rows: a hypothesis that ended, a slot that is
free.  What they hold, short lengths, no pages, pages that others have by now, is not read."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
from ops_ref import Batch  # noqa: E402
from test_gpu_kv_prefix import _check, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def _idle(b, first, last, how):
    """What the sequences first .. last - 1 hold."""
    for s in range(first, last):
        if how == "short":
            b.length[s] = 3
        elif how == "none":
            b.length[s] = 0
            b.table[s] = -1
        else:  # the last sequence's pages, in another order
            b.table[s] = b.table[-1][::-1]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("how", ["short", "none", "taken"])
@pytest.mark.parametrize("new", [[0, 1, 1, 1], [0, 0, 1, 0, 2], [0, 30, 0, 41], [0, 0, 0, 1]])
@pytest.mark.parametrize("dim,heads", [(64, (4, 2)), (128, (8, 2))])
def test_first_of_a_group(mit2, ctx, dtype, how, new, dim, heads):  # noqa: F811
    b = Batch(new, [150 + 7 * s + n for s, n in enumerate(new)], page=16, dim=dim, q_heads=heads[0], kv_heads=heads[1], dtype=dtype, seed=21)
    lead = next(s for s, n in enumerate(new) if n)
    context_ref.share(b, [lead, len(new)], [140], True)
    _idle(b, 0, lead, how)
    _check(mit2, ctx, b, [0, len(new)], [140], made=True, what=f"{dtype} {how} {new}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", ["short", "none", "taken"])
@pytest.mark.parametrize("idle", [1, 63, 64, 130])
def test_of_many_sequences_and_groups(mit2, ctx, dtype, how, idle):  # noqa: F811
    """More sequences than a wave's lanes; a group without new rows; a second group right behind the first's idle ones."""
    new = [1, 2] + [0] * idle + [1] * 20 + [0] * 3 + [0] + [3, 1]
    b = Batch(new, [100 + 5 * (s % 9) + n for s, n in enumerate(new)], page=8, dim=64, q_heads=2, kv_heads=1, dtype=dtype, seed=idle, lead_rows=2, tail_rows=1)
    lead, end = 2 + idle, 2 + idle + 20
    context_ref.share(b, [lead, end], [96], True)
    context_ref.share(b, [end + 4, end + 6], [88], True)
    _idle(b, 2, lead, how)
    _idle(b, end, end + 4, how)
    _check(mit2, ctx, b, [2, end, end + 3, end + 6], [96, 96, 88], made=True, what=f"{dtype} {how} {idle}")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_shared_rows_of_the_first_that_has_new_ones(mit2, ctx, dtype):  # noqa: F811
    """The bound is of the sequences with new rows: all 140 rows, though the first, without any, has 10."""
    b = Batch([0, 1, 1], [10, 150, 151], page=16, dim=64, dtype=dtype, seed=7)
    context_ref.share(b, [1, 3], [140], False)
    _check(mit2, ctx, b, [0, 3], [140], made=True, hint=150)
