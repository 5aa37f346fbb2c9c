"""Values that are not finite and that rows do see, in attention with shared prefixes (mit2cfm_kv_prefix_attention_device): a shared row is seen by
every new row of its group, a cached row of a sequence's own by every new row of it, a new row by those that its mask says."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
import ops_ref  # noqa: E402
from context_ref import mine  # noqa: E402
from ops_ref import Batch  # noqa: E402
from test_gpu_kv_prefix import Shared, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# dim, heads, new rows: one query tile a wave, two, the block form by its groups and by its sequences
FORMS = [(64, (2, 2), [1, 1, 1]), (64, (2, 1), [1] * 20), (96, (4, 4), [20, 14, 1]), (64, (3, 3), [1] * 35), (128, (8, 2), [1] * 7), (128, (8, 2), [12, 9, 1]),
         (64, (2, 2), [70, 1, 40]), (64, (2, 2), [230, 1]), (128, (8, 2), [170, 3])]
SHARED, PAGE = 328, 16


def _batch(new, heads, dim, dtype):
    b = Batch(new, [SHARED + n + 40 + 9 * (s % 5) for s, n in enumerate(new)], page=PAGE, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim,
              lead_rows=1, tail_rows=2)
    context_ref.share(b, [0, len(new)], [SHARED], True)
    return b


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new", FORMS)
@pytest.mark.parametrize("tree", [False, True])
def test_cached_rows(mit2, ctx, dtype, dim, heads, new, tree):  # noqa: F811
    """NaN, an infinity, two that meet, in a shared row and in a sequence's own: all that see them have them, no other element changes by a bit."""
    b = _batch(new, heads, dim, dtype)
    mask = ops_ref.trees(b, 17)[0] if tree else None
    bounds, said, last = [0, len(new)], [SHARED], len(new) - 1
    clean = Shared(mit2, b, bounds, said, mask=mask).run(ctx)
    odd = (2, 5, 9, dim - 1)
    rest = [d for d in range(dim) if d not in odd]
    values = b.v.clone()
    for seq, place, rows in ((0, 0, mine(b)), (0, 200, mine(b)), (0, 319, mine(b)),  # (whole pages: of all)
                             (last, SHARED + 20, None), (last, b.length[last] - new[last] - 1, None)):
        if rows is None:
            rows = torch.zeros(b.rows, dtype=torch.bool)
            rows[int(b.start[seq]): int(b.start[seq + 1])] = True
        b.v = values.clone()
        at, also = (b.v[b.page_of(seq, j), :, j % PAGE] for j in (place, place - 1 if place else 1))
        at[:, 5], at[:, 9], at[:, dim - 1], at[:, 2], also[:, 2] = math.nan, math.inf, -math.inf, math.inf, -math.inf
        got = Shared(mit2, b, bounds, said, mask=mask).run(ctx)
        m = mine(b)
        assert torch.equal(got[m][:, :, rest], clean[m][:, :, rest]), place
        assert torch.equal(got[m & ~rows], clean[m & ~rows]), place
        assert bool(torch.isnan(got[rows][:, :, 5]).all()) and bool(torch.isnan(got[rows][:, :, 2]).all()), place
        assert bool((got[rows][:, :, 9] == math.inf).all()) and bool((got[rows][:, :, dim - 1] == -math.inf).all()), place


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new", [x for x in FORMS if max(x[2]) > 1])
def test_new_rows_beside_cached_ones(mit2, ctx, dtype, dim, heads, new):  # noqa: F811
    """An infinity and a NaN in a new row reach the rows that see it, and an infinity of a shared row in the same call all."""
    b = _batch(new, heads, dim, dtype)
    bounds, said = [0, len(new)], [SHARED]
    clean = Shared(mit2, b, bounds, said).run(ctx)
    i, old = new[0] // 2, b.length[0] - new[0]
    j = old + i
    b.v[b.page_of(0, j), :, j % PAGE, 7] = math.inf
    b.v[b.page_of(0, j), :, j % PAGE, 8] = math.nan
    b.v[b.page_of(0, 3), :, 3, 11] = -math.inf
    got = Shared(mit2, b, bounds, said).run(ctx)
    m = mine(b)
    see = torch.zeros(b.rows, dtype=torch.bool)
    see[int(b.start[0]) + i: int(b.start[1])] = True
    assert bool((got[see][:, :, 7] == math.inf).all()) and bool(torch.isnan(got[see][:, :, 8]).all())
    assert torch.equal(got[m & ~see][:, :, 7:9], clean[m & ~see][:, :, 7:9])
    assert bool((got[m][:, :, 11] == -math.inf).all())
    rest = [d for d in range(dim) if d not in (7, 8, 11)]
    assert torch.equal(got[m][:, :, rest], clean[m][:, :, rest])
