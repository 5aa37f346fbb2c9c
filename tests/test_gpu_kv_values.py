"""Values of the paged cache that are not finite and that a row does see (mit2cfm_kv_attention_device): a cached row before the
new ones is seen by every row of its sequence, wherever it lies beside the tiles, the new rows and the entries that are no page."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ops_ref  # noqa: E402
from ops_ref import Batch  # noqa: E402
from test_gpu_kv_ops import On, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# one query tile a wave, two, the block form (by the rows a sequence and the head size)
FORMS = [(64, (2, 2), [1, 1], 2), (128, (8, 2), [2, 3], 1), (64, (2, 1), [12, 14], 2), (96, (4, 4), [40, 30], 1), (64, (2, 2), [100, 60], 1),
         (128, (8, 2), [60, 70], 1)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new,page_step", FORMS)
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("hole", [False, True])
def test_a_cached_row_s_values_reach_every_row_of_its_sequence(mit2, ctx, dtype, dim, heads, new, page_step, tree, hole):  # noqa: F811
    """NaN and both infinities in cached rows before the new ones: in the first tile, in the middle, right before the new rows (in one tile with
    them), with and without an entry that is no page before them.  No other element changes by a bit."""
    for page, old in ((16, (705, 330)), (64 * page_step, (687, 97))):
        b = Batch(new, [n + o for n, o in zip(new, old)], page=page, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim + page)
        mask = ops_ref.trees(b, 17)[0] if tree else None
        if hole:
            b.table[0, 1], b.table[1, 0] = -1, b.pages
        clean = On(mit2, b).attend(ctx, mask=mask)
        gone = {s: {j for j in range(b.length[s]) if b.page_of(s, j) < 0} for s in range(2)}
        for where in ((3, 1), (old[0] // 2, old[1] // 2), (old[0] - 15, old[1] - 1), (old[0] - 1, old[1] - 20)):
            b2 = Batch(new, b.length, page=page, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim + page)
            b2.table[:] = b.table
            hit = [j not in gone[s] for s, j in enumerate(where)]
            for s, j in enumerate(where):
                if hit[s]:
                    for d, value in ((5, math.nan), (9, math.inf), (dim - 1, -math.inf)):
                        b2.v[b2.page_of(s, j), :, j % page, d] = value
            got = On(mit2, b2).attend(ctx, mask=mask)
            rest = [d for d in range(dim) if d not in (5, 9, dim - 1)]
            assert torch.equal(got[:, :, rest], clean[:, :, rest]), where
            for s in range(2):
                mine = slice(int(b.start[s]), int(b.start[s + 1]))
                if hit[s]:
                    assert bool(torch.isnan(got[mine, :, 5]).all()), (where, s)
                    assert bool((got[mine, :, 9] == math.inf).all()) and bool((got[mine, :, dim - 1] == -math.inf).all()), (where, s)
                else:
                    assert torch.equal(got[mine], clean[mine])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("new,heads,dim", [([1], (1, 1), 64), ([70], (2, 2), 64), ([70], (4, 1), 128)])
def test_values_beside_the_new_rows_of_a_long_cache(mit2, ctx, dtype, new, heads, dim):  # noqa: F811
    """The same where the keys are split over blocks: a NaN in each of the last 40 cached rows before the new ones, one at a time; and a new
    row's NaN beside a cached row's infinity reaches the rows that see it, and the infinity all."""
    b = Batch(new, [3001 + new[0]], page=32, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=4)
    v = b.v.clone()
    for back in range(1, 41):
        j = 3001 - back
        b.v = v.clone()
        b.v[b.page_of(0, j), :, j % b.page, 2] = math.nan
        got = On(mit2, b).attend(ctx)
        assert bool(torch.isnan(got[:, :, 2]).all()) and bool(torch.isfinite(got[:, :, 3:]).all()), back
    b.v = v.clone()
    i = new[0] // 2
    b.v[b.page_of(0, 3001 + i), :, (3001 + i) % b.page, 7] = math.nan
    b.v[b.page_of(0, 2999), :, 2999 % b.page, 8] = -math.inf
    got = On(mit2, b).attend(ctx)
    assert bool(torch.isnan(got[i:, :, 7]).all()) and bool(torch.isfinite(got[:i, :, 7]).all())
    assert bool((got[:, :, 8] == -math.inf).all()) and bool(torch.isfinite(got[:, :, 9:]).all())
