"""The added-up attention weights (mit2cfm_kv_weigh_device) on the GPU against a plain 64-bit restatement (context_ref.py)."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
import ops_ref  # noqa: E402
from context_ref import DEV, On, check  # noqa: E402
from ops_ref import TORCH, Batch  # noqa: E402

pytestmark = pytest.mark.gpu
LENGTHS = [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300]


@pytest.fixture(scope="module")
def ctx(mit2):
    c = mit2.Context(synthetic_seed=3, device=0)
    yield c
    c.close()


class Weigh:
    """A call's buffers: weights as they were, NaN where nothing may be written."""

    def __init__(self, mit2, b, *, scale=None, mask=None, decay=1.0, last=0, stride=None, lse=None, in_place=False, position=None, born=False, seed=1):
        self.on, self.b, self.mask, self.decay, self.last = On(mit2, b), b, mask, decay, last
        self.scale = b.dim ** -0.5 if scale is None else scale
        self.lse = (context_ref.lse64(b, self.scale, mask) if lse is None else lse).float()
        stride = stride or b.table.shape[1] * b.page
        g = torch.Generator().manual_seed(seed)
        self.weights = torch.rand(len(b.new), b.kv_heads, stride, generator=g) * 3
        self.dev_weights = self.weights.to(DEV)
        self.out = self.dev_weights if in_place else torch.full_like(self.dev_weights, math.nan)
        self.dev_lse = self.lse.to(DEV)
        self.dev_mask = None if mask is None else torch.from_numpy(mask.view(np.int32)).to(DEV)
        self.born = torch.full(self.weights.shape, -7, dtype=torch.int32, device=DEV) if born else None
        self.position = None if position is None else torch.as_tensor(position, dtype=torch.int32, device=DEV)
        d = b.dim
        self.args = mit2.KvWeigh(q=self.on.q.data_ptr(), q_row=b.q_heads * d, q_head=d, q_heads=b.q_heads, scale=self.scale,
                                 mask=None if mask is None else self.dev_mask.data_ptr(), mask_words=0 if mask is None else mask.shape[1],
                                 last_rows=last, lse=self.dev_lse.data_ptr(), weights=self.dev_weights.data_ptr(), weights_out=self.out.data_ptr(),
                                 weight_stride=stride, decay=decay, position=None if position is None else self.position.data_ptr(),
                                 born=self.born.data_ptr() if born else None)

    def run(self, ctx):
        torch.cuda.synchronize()
        ctx.kv_weigh_device(self.on.cache, self.on.rows, self.args, sync=True)
        return self.out.double().cpu()

    def check(self, ctx, what=""):
        raw = self.run(ctx)
        got = raw.clone()
        ref, tol = context_ref.weigh64(self.b, self.lse, self.weights, self.scale, self.mask, self.decay, self.last)
        b = self.b
        in_place = self.out is self.dev_weights
        for s, n in enumerate(b.new):  # what is left alone
            places = max(0, min(b.length[s], ref.shape[2], b.table.shape[1] * b.page)) if n else 0
            if not in_place:
                assert bool(torch.isnan(got[s, :, places:]).all()), "places past the end were written"
                got[s, :, places:] = ref[s, :, places:] = 0.0
        check(got, ref, tol, what or f"{b.dtype} dim {b.dim} heads {b.q_heads}/{b.kv_heads} page {b.page}")
        return raw


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,q_heads,kv_heads", [(64, 20, 20), (128, 8, 2), (32, 7, 1), (96, 6, 1), (192, 4, 2), (256, 3, 1), (128, 16, 1), (64, 34, 2)])
def test_single_tokens(mit2, ctx, dtype, dim, q_heads, kv_heads):
    b = Batch([1] * len(LENGTHS), LENGTHS, page=16, kv_heads=kv_heads, q_heads=q_heads, dim=dim, dtype=dtype, seed=dim)
    Weigh(mit2, b).check(ctx)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new", [(64, (4, 4), [33, 1, 0, 64, 7, 90]), (128, (8, 2), [17, 40, 3, 0, 9, 65]), (96, (5, 1), [2, 3, 1, 1, 0, 4]),
                                           (256, (2, 1), [70, 5, 0, 3, 1, 9])])
@pytest.mark.parametrize("tree", [False, True])
def test_chains_and_trees(mit2, ctx, dtype, dim, heads, new, tree):
    b = Batch(new, [n + (0, 50, 9, 130, 1, 257)[s] for s, n in enumerate(new)], page=16, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype,
              seed=dim, tail_rows=2, lead_rows=3)
    Weigh(mit2, b, mask=ops_ref.trees(b, dim)[0] if tree else None, decay=0.75).check(ctx)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads", [(32, (6, 2)), (64, (3, 3)), (96, (8, 1)), (128, (5, 1)), (192, (2, 1)), (256, (14, 2))])
@pytest.mark.parametrize("tree", [False, True])
def test_prompts(mit2, ctx, dtype, dim, heads, tree):
    """Queries of many tiles; a page is missing, of one sequence the rows are more than its length."""
    new = [131, 0, 200, 97]
    b = Batch(new, [131 + 300, 50, 200, 97 + 65], page=16, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim, tail_rows=1, lead_rows=2)
    b.table[0, 2] = -1
    b.length[2] = 190
    Weigh(mit2, b, mask=ops_ref.trees(b, dim)[0] if tree else None, decay=0.75).check(ctx)


@pytest.mark.parametrize("dtype,dim,last", [("f32", 64, 0), ("f16", 128, 0), ("bf16", 96, 0), ("f16", 64, 7)])
def test_many_sequences_of_some_rows(mit2, ctx, dtype, dim, last):
    new = [(37 * s) % 41 for s in range(50)]
    b = Batch(new, [n + (29 * s) % 300 for s, n in enumerate(new)], page=8, q_heads=12, kv_heads=4, dim=dim, dtype=dtype, seed=dim)
    Weigh(mit2, b, decay=0.5, last=last).check(ctx)


@pytest.mark.parametrize("last", [1, 5, 16, 40, 1000])
@pytest.mark.parametrize("tree", [False, True])
def test_last_rows_alone(mit2, ctx, last, tree):
    b = Batch([60, 3, 0, 130], [300, 3, 8, 131], page=32, q_heads=4, kv_heads=2, dim=64, dtype="bf16", seed=last, lead_rows=1)
    Weigh(mit2, b, mask=ops_ref.trees(b, 4)[0] if tree else None, last=last).check(ctx, f"last {last}")


@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0, -1.5])
@pytest.mark.parametrize("in_place", [False, True])
def test_decay_and_in_place(mit2, ctx, decay, in_place):
    b = Batch([1, 0, 20], [100, 7, 90], page=8, dim=64, dtype="f32", seed=3)
    Weigh(mit2, b, decay=decay, in_place=in_place).check(ctx, f"decay {decay}")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page", [1, 2, 8, 128, 1024])
def test_pages(mit2, ctx, dtype, page):
    b = Batch([1, 3, 0, 20], [90, 131, 0, 57], page=page, dim=64, dtype=dtype, seed=page, lead_rows=1, tail_rows=2)
    Weigh(mit2, b).check(ctx)


@pytest.mark.parametrize("new", [[1, 1, 2], [30, 60, 2]])
def test_missing_pages_and_odd_lengths(mit2, ctx, new):
    b = Batch(new, [100, 77, 40], page=16, dim=64, dtype="f16", seed=10)
    b.table[0, 0], b.table[0, 3], b.table[1, 4], b.table[2, 1] = -1, b.pages, 2 ** 31 - 1, -2 ** 31
    Weigh(mit2, b).check(ctx)
    b.length = [b.table.shape[1] * 16 + 9, 77, new[2] - 1]  # past the table; fewer rows than new ones
    Weigh(mit2, b).check(ctx)
    b.length = [0, -5, 40]
    Weigh(mit2, b).check(ctx)


@pytest.mark.parametrize("stride", [1, 63, 100, 400])
def test_strides_of_the_weights(mit2, ctx, stride):
    b = Batch([1, 40], [130, 90], page=16, dim=64, dtype="bf16", seed=5)
    Weigh(mit2, b, stride=stride, born=True).check(ctx)


@pytest.mark.parametrize("new", [1, 25])
def test_rows_that_see_nothing_add_nothing(mit2, ctx, new):
    b = Batch([new, new], [new, 60], page=16, dim=64, dtype="f32", seed=6)
    mask = ops_ref.trees(b, 3)[0]
    mask[0] = 0
    w = Weigh(mit2, b, mask=mask)
    assert bool((w.lse[0] == -math.inf).all())
    w.check(ctx)
    # rows that see keys, said to see nothing
    lse = w.lse.clone()
    lse[-1] = -math.inf
    Weigh(mit2, b, mask=mask, lse=lse).check(ctx)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [2, 30])
def test_what_is_not_finite_stays_in_its_place(mit2, ctx, dtype, new):
    b = Batch([new, 1], [90, 40], page=16, dim=64, dtype=dtype, seed=8)
    w = Weigh(mit2, b)
    clean = w.check(ctx)
    used = np.zeros((b.pages, b.page), bool)
    for s, n in enumerate(b.length):
        for j in range(n):
            used[b.page_of(s, j), j % b.page] = True
    b.k.permute(0, 2, 1, 3)[torch.from_numpy(~used)] = math.nan
    b.k[b.page_of(0, 33), :, 33 % b.page, 7] = math.nan  # a cached row that all see
    b.k[b.page_of(0, 89), :, 89 % b.page, 0] = math.inf  # the last new row: seen by itself
    got = Weigh(mit2, b, lse=w.lse).run(ctx)
    assert bool(torch.isnan(got[0, :, 33]).all())
    for x in (got, clean):
        x[0, :, 33] = x[0, :, 89] = 0.0
    assert torch.equal(got.nan_to_num(-1.0), clean.nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_large_and_equal_scores(mit2, ctx, dtype):
    b = Batch([1, 4, 40], [300, 90, 60], dim=64, dtype=dtype, seed=11)
    b.q *= 8
    b.k *= 4
    for scale in (1.0, 0.0, -0.25):
        Weigh(mit2, b, scale=scale).check(ctx, f"{dtype} scale {scale}")


@pytest.mark.parametrize("new", [3, 40])
def test_births(mit2, ctx, new):
    b = Batch([new, 0, 2], [90, 10, 2], page=16, dim=64, dtype="f16", seed=12, lead_rows=2, tail_rows=1)
    position = np.arange(b.rows, dtype=np.int32) * 3 + 1000
    for where in (None, position):
        w = Weigh(mit2, b, born=True, position=where)
        w.check(ctx)
        want = torch.full(w.weights.shape, -7, dtype=torch.int32)
        for row, s, i, before in b.each_row():
            want[s, :, before + i] = before + i if where is None else int(position[row])
        assert torch.equal(w.born.cpu(), want)


def test_strides_of_the_queries(mit2, ctx):
    b = Batch([1, 33], [60, 200], q_heads=4, kv_heads=2, dim=64, dtype="f16", seed=12)
    ref = Weigh(mit2, b).check(ctx)
    w = Weigh(mit2, b)
    width = b.q_heads * b.dim + 5
    q = torch.zeros(b.rows * width + 1, dtype=TORCH["f16"], device=DEV)
    q[1:].view(b.rows, width)[:, : b.q_heads * b.dim] = w.on.q.reshape(b.rows, -1)
    w.args.q, w.args.q_row = q.data_ptr() + 2, width
    assert torch.equal(w.run(ctx).nan_to_num(-1.0), ref.nan_to_num(-1.0))


@pytest.mark.parametrize("new", [1, 50])
def test_hints_and_the_same_bits(mit2, ctx, new):
    b = Batch([new, 1], [2000, 70], dim=64, dtype="bf16", seed=13)
    first = Weigh(mit2, b).check(ctx)
    for hint in (0, 1, 100, 1 << 20, 2 ** 32 - 1):
        w = Weigh(mit2, b)
        w.on.rows.max_length = hint
        assert torch.equal(w.run(ctx).nan_to_num(-1.0), first.nan_to_num(-1.0))


def test_many_sequences(mit2, ctx):
    new = [(s % 3) for s in range(300)]
    b = Batch(new, [n + (11 * s) % 50 for s, n in enumerate(new)], page=8, kv_heads=1, q_heads=2, dim=32, dtype="f16", seed=9, tail_rows=5)
    Weigh(mit2, b).check(ctx)


@pytest.mark.parametrize("seqs", [0, 2])
def test_nothing_to_do(mit2, ctx, seqs):
    b = Batch([1, 1], [4, 4], dim=64, dtype="f32", seed=15)
    w = Weigh(mit2, b)
    w.on.rows.seqs, w.on.rows.rows = seqs, 0 if seqs else 2
    assert bool(torch.isnan(w.run(ctx)).all())


def test_offsets_past_32_bits(mit2, ctx):
    """Keys in the last pages of a cache of over 2^32 elements; weights over 2^31 elements in."""
    pages, heads, page, dim = 70000, 8, 64, 128
    b = Batch([1, 3], [100, 40], page=page, kv_heads=heads, q_heads=heads, dim=dim, dtype="bf16", seed=16)
    w = Weigh(mit2, b)
    ref = w.check(ctx)
    flat = torch.empty(pages * heads * page * dim, dtype=torch.bfloat16, device=DEV)
    far = torch.empty((heads + 1) * (1 << 28) + 1000, device=DEV)
    try:
        shift = pages - b.pages
        flat.view(pages, heads, page, dim)[shift:] = w.on.k
        w.on.table += shift * (w.on.table >= 0)
        w.on.cache.k, w.on.cache.v, w.on.cache.pages = flat.data_ptr(), flat.data_ptr(), pages
        stride = 1 << 28
        b2 = w.weights.shape[2]
        for h in range(heads):
            far[h * stride: h * stride + b2] = w.dev_weights[0, h]
        w.on.rows.seqs = 1  # (the first sequence's eight heads)
        w.args.weights = w.args.weights_out = far.data_ptr()
        w.args.weight_stride = stride
        torch.cuda.synchronize()
        ctx.kv_weigh_device(w.on.cache, w.on.rows, w.args, sync=True)
        for h in range(heads):
            assert torch.equal(far[h * stride: h * stride + 100].double().cpu(), ref[0, h, :100])
    finally:
        del flat, far
        torch.cuda.empty_cache()
