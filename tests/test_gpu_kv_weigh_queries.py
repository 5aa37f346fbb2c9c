"""The added-up attention weights (mit2cfm_kv_weigh_device) where a block's waves share their keys and divide the queries, against the plain 64-bit
restatement (context_ref.py); test_weigh_plan.py holds these sizes to that form."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ops_ref  # noqa: E402
import weigh_cases as cases  # noqa: E402
from context_ref import DEV, check, weigh64  # noqa: E402
from ops_ref import TORCH, Batch  # noqa: E402
from test_gpu_kv_weigh import Weigh, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def _name(c):
    a = c["args"]
    return f"{a['dtype']}-{a['dim']}-{a['q_heads']}x{a['kv_heads']}-{len(a['new'])}"


def _batch(c):
    return Batch(**c["args"], seed=c["args"]["dim"])


@pytest.mark.parametrize("c", cases.SIZES, ids=_name)
@pytest.mark.parametrize("tree", [False, True])
def test_types_and_sizes(mit2, ctx, c, tree):  # noqa: F811
    b = _batch(c)
    Weigh(mit2, b, mask=ops_ref.trees(b, b.dim)[0] if tree else None, decay=0.75).check(ctx)


@pytest.mark.parametrize("c", cases.BIRTHS, ids=_name)
@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("cut", [False, True])
def test_births(mit2, ctx, c, positions, cut):  # noqa: F811
    """New rows' places get their positions or places, all others keep theirs; cut: the lines end inside the new rows."""
    b = _batch(c)
    position = np.arange(b.rows, dtype=np.int32) * 3 - 1000 if positions else None
    w = Weigh(mit2, b, born=True, position=position, stride=max(b.length) - 50 if cut else None)
    w.check(ctx)
    want = torch.full(w.weights.shape, -7, dtype=torch.int32)
    for row, s, i, before in b.each_row():
        if before + i < want.shape[2]:
            want[s, :, before + i] = before + i if position is None else int(position[row])
    assert torch.equal(w.born.cpu(), want)


@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0, -1.5])
@pytest.mark.parametrize("in_place", [False, True])
def test_decay_and_in_place(mit2, ctx, decay, in_place):  # noqa: F811
    Weigh(mit2, _batch(cases.OTHERS["in_place"]), decay=decay, in_place=in_place, born=True).check(ctx, f"decay {decay}")


@pytest.mark.parametrize("stride,c", cases.STRIDES, ids=lambda x: _name(x) if isinstance(x, dict) else str(x))
def test_strides_of_the_weights(mit2, ctx, stride, c):  # noqa: F811
    Weigh(mit2, _batch(c), stride=stride, born=True).check(ctx, f"stride {stride}")


@pytest.mark.parametrize("c", cases.XCD, ids=_name)
@pytest.mark.parametrize("last", [0, 50])
def test_lines_by_xcds(mit2, ctx, c, last):  # noqa: F811
    Weigh(mit2, _batch(c), decay=0.5, last=last, born=True).check(ctx)


@pytest.mark.parametrize("tree", [False, True])
def test_last_rows_alone(mit2, ctx, tree):  # noqa: F811
    b = _batch(cases.OTHERS["last"])
    Weigh(mit2, b, mask=ops_ref.trees(b, 4)[0] if tree else None, last=cases.LAST).check(ctx)


def test_missing_pages_and_odd_lengths(mit2, ctx):  # noqa: F811
    b = _batch(cases.OTHERS["odd_places"])
    b.table[0, 0], b.table[0, 3], b.table[1, 4], b.table[2, 1] = -1, b.pages, 2 ** 31 - 1, -2 ** 31
    Weigh(mit2, b).check(ctx)
    b.length = [b.table.shape[1] * 16 + 9, b.length[1], b.new[2] - 1]  # past the table; fewer rows than new ones
    Weigh(mit2, b).check(ctx)
    b.length = [0, -5, b.length[2]]
    Weigh(mit2, b).check(ctx)


def test_rows_that_see_nothing_add_nothing(mit2, ctx):  # noqa: F811
    b = _batch(cases.OTHERS["unseen"])
    mask = ops_ref.trees(b, 3)[0]
    mask[[0, 1, 17, 40, 109]] = 0
    w = Weigh(mit2, b, mask=mask)
    assert bool((w.lse[[0, 1, 17, 40, 109]] == -math.inf).all())
    w.check(ctx)
    lse = w.lse.clone()  # rows that see keys, said to see nothing
    lse[-1] = lse[140] = -math.inf
    Weigh(mit2, b, mask=mask, lse=lse).check(ctx)


def test_large_and_equal_scores(mit2, ctx):  # noqa: F811
    b = _batch(cases.OTHERS["large"])
    b.q *= 8
    b.k *= 4
    for scale in (1.0, 0.0, -0.25):
        Weigh(mit2, b, scale=scale).check(ctx, f"scale {scale}")


@pytest.mark.parametrize("c", cases.FINITE, ids=_name)
def test_what_is_not_finite_stays_in_its_place(mit2, ctx, c):  # noqa: F811
    b = _batch(c)
    w = Weigh(mit2, b)
    clean = w.check(ctx)
    used = np.zeros((b.pages, b.page), bool)
    for s, n in enumerate(b.length):
        for j in range(n):
            used[b.page_of(s, j), j % b.page] = True
    b.k.permute(0, 2, 1, 3)[torch.from_numpy(~used)] = math.nan
    last = b.length[0] - 1
    b.k[b.page_of(0, 33), :, 33 % b.page, 7] = math.nan  # a cached row that all see
    b.k[b.page_of(0, last), :, last % b.page, 0] = math.inf  # the last new row: seen by itself
    got = Weigh(mit2, b, lse=w.lse).run(ctx)
    assert bool(torch.isnan(got[0, :, 33]).all())
    for x in (got, clean):
        x[0, :, 33] = x[0, :, last] = 0.0
    assert torch.equal(got.nan_to_num(-1.0), clean.nan_to_num(-1.0))
    # a log sum that is NaN reaches the keys that its row sees, one of +inf adds nothing
    lse = w.lse.clone()
    lse[5] = math.inf
    plain = Weigh(mit2, b, lse=lse).run(ctx)
    lse[100] = math.nan  # row 100 of the first sequence sees its places up to before + 100
    got = Weigh(mit2, b, lse=lse).run(ctx)
    see = b.length[0] - b.new[0] + 100 + 1
    assert bool(torch.isnan(got[0, :, :see]).all())
    for x in (got, plain):
        x[0, :, :see] = x[0, :, last] = 0.0
    assert torch.equal(got.nan_to_num(-1.0), plain.nan_to_num(-1.0))


@pytest.mark.parametrize("c", cases.QUERIES, ids=_name)
def test_strides_of_the_queries(mit2, ctx, c):  # noqa: F811
    """Queries in a projection's rows at an odd stride, element by element: not by way of LDS."""
    b = _batch(c)
    w = Weigh(mit2, b)
    width = b.q_heads * b.dim + 5
    q = torch.zeros(b.rows * width + 1, dtype=TORCH[b.dtype], device=DEV)
    q[1:].view(b.rows, width)[:, : b.q_heads * b.dim] = w.on.q.reshape(b.rows, -1)
    w.args.q, w.args.q_row = q.data_ptr() + q.element_size(), width
    w.check(ctx)


def test_hints(mit2, ctx):  # noqa: F811
    """Shorter ones give a block several runs of keys, longer ones blocks without any."""
    b = _batch(cases.LONG)
    first = Weigh(mit2, b, born=True).check(ctx)
    for hint in (0, 1, 100, 1 << 20, 2 ** 32 - 1):
        w = Weigh(mit2, b, born=True)
        w.on.rows.max_length = hint
        assert torch.equal(w.run(ctx).nan_to_num(-1.0), first.nan_to_num(-1.0))


@pytest.mark.parametrize("c", cases.HINTED, ids=_name)
def test_hints_that_choose_the_form(mit2, ctx, c):  # noqa: F811
    """Any hint is right; where hints choose another form its sums go in another order, and bits are each form's own, the same each time."""
    b = _batch(c)
    ref, tol = None, None
    for hints in (cases.FEW, cases.MANY):
        first = None
        for hint in hints:
            w = Weigh(mit2, b)
            w.on.rows.max_length = hint
            raw = w.run(ctx)
            if ref is None:
                ref, tol = weigh64(b, w.lse, w.weights, w.scale)
                for s, n in enumerate(b.length):
                    ref[s, :, n:] = 0.0
            if first is None:
                first = raw
            assert torch.equal(raw.nan_to_num(-1.0), first.nan_to_num(-1.0)) and torch.equal(w.run(ctx).nan_to_num(-1.0), first.nan_to_num(-1.0))
        got = first.clone()
        for s, n in enumerate(b.length):
            assert bool(torch.isnan(got[s, :, n:]).all())
            got[s, :, n:] = 0.0
        check(got, ref, tol, f"hints {hints}")


def test_offsets_past_32_bits(mit2, ctx):  # noqa: F811
    """Keys in the last pages of a cache of over 2^32 elements, queries and weights over 2^31 elements in."""
    pages, heads, page, dim, new = 70000, 8, 64, 128, 130
    b = Batch([new], [new + 200], page=page, kv_heads=heads, q_heads=heads, dim=dim, dtype="bf16", seed=16)
    w = Weigh(mit2, b)
    flat = torch.empty(pages * heads * page * dim, dtype=torch.bfloat16, device=DEV)
    stride, width = 1 << 28, 17 << 20
    far, q = torch.empty(heads * stride, device=DEV), torch.zeros((new - 1) * width + heads * dim, dtype=torch.bfloat16, device=DEV)
    try:
        shift = pages - b.pages
        flat.view(pages, heads, page, dim)[shift:] = w.on.k
        w.on.table += shift * (w.on.table >= 0)
        w.on.cache.k, w.on.cache.v, w.on.cache.pages = flat.data_ptr(), flat.data_ptr(), pages
        for i in range(new):
            q[i * width: i * width + heads * dim] = w.on.q[i].reshape(-1)
        w.args.q, w.args.q_row = q.data_ptr(), width
        n = b.length[0]
        for h in range(heads):
            far[h * stride: h * stride + n] = w.dev_weights[0, h, :n]
        w.args.weights = w.args.weights_out = far.data_ptr()
        w.args.weight_stride = stride
        torch.cuda.synchronize()
        ctx.kv_weigh_device(w.on.cache, w.on.rows, w.args, sync=True)
        ref, tol = weigh64(b, w.lse, w.weights, w.scale)
        got = torch.stack([far[h * stride: h * stride + n] for h in range(heads)]).double().cpu()
        check(got, ref[0, :, :n], tol[0, :, :n], "far pages")
    finally:
        del flat, far, q
        torch.cuda.empty_cache()
