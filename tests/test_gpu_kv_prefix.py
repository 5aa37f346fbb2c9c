"""Attention of sequences that share their first rows (mit2cfm_kv_prefix_attention_device) on the GPU against the plain 64-bit
attention (ops_ref.py), with its log sums."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
import ops_ref  # noqa: E402
from context_ref import DEV, On, check, mine  # noqa: E402
from ops_ref import TORCH, Batch  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(mit2):
    c = mit2.Context(synthetic_seed=3, device=0)
    yield c
    c.close()


class Shared:
    """A call's buffers."""

    def __init__(self, mit2, b, bounds, shared, *, mask=None, scale=None, hint=None, lse=True):
        self.on, self.b, self.mask = On(mit2, b), b, mask
        self.scale = b.dim ** -0.5 if scale is None else scale
        self.args = self.on.attention_args(scale=scale, mask=mask)
        self.bounds, self.shared = (torch.tensor(list(x) or [0], dtype=torch.int32, device=DEV) for x in (bounds, shared))
        self.lse = torch.full((b.rows, b.q_heads), math.nan, device=DEV)
        self.prefix = mit2.KvPrefix(group=self.bounds.data_ptr(), shared=self.shared.data_ptr(), groups=len(shared),
                                    max_shared=max(list(shared) + [0]) if hint is None else hint, lse=self.lse.data_ptr() if lse else None)
        self.mit2 = mit2

    def run(self, ctx):
        n = self.mit2.kv_prefix_attention_workspace(self.on.cache, self.on.rows, self.b.q_heads, self.prefix)
        self.workspace = torch.full((n + 256,), 255, dtype=torch.uint8, device=DEV)  # (NaN, were it read before it is written)
        self.args.workspace, self.args.workspace_bytes = self.workspace.data_ptr(), n
        torch.cuda.synchronize()
        ctx.kv_prefix_attention_device(self.on.cache, self.on.rows, self.args, self.prefix, sync=True)
        assert bool((self.workspace[n:] == 255).all())
        return self.on.out.double().cpu()


def _check(mit2, ctx, b, bounds, shared, *, alias=True, mask=None, scale=None, hint=None, what="", made=False):
    if not made:
        context_ref.share(b, bounds, shared, alias)
    x = Shared(mit2, b, bounds, shared, mask=mask, scale=scale, hint=hint)
    got = x.run(ctx)
    ref, tol = ops_ref.attention64(b, x.scale, mask)
    m = mine(b)
    what = what or f"{b.dtype} dim {b.dim} heads {b.q_heads}/{b.kv_heads} page {b.page}"
    lse = x.lse.double().cpu()
    assert bool(torch.isnan(got[~m]).all()) and bool(torch.isnan(lse[~m]).all()), "rows of no sequence were written"
    check(got[m], ref[m], tol[m], what)
    check(lse[m], context_ref.lse64(b, x.scale, mask)[m], context_ref.lse_tolerance(b, x.scale, mask)[m], "lse " + what)
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,q_heads,kv_heads", [(64, 20, 20), (128, 8, 2), (32, 7, 1), (96, 6, 1), (192, 4, 2), (256, 3, 1), (128, 16, 1), (64, 34, 2)])
def test_single_tokens(mit2, ctx, dtype, dim, q_heads, kv_heads):
    lens = [201, 202, 300, 217, 330, 260, 64, 70, 66]
    b = Batch([1] * 9, lens, page=16, kv_heads=kv_heads, q_heads=q_heads, dim=dim, dtype=dtype, seed=dim)
    _check(mit2, ctx, b, [0, 6, 9], [200, 63])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 1, 63, 64, 65, 127, 128, 200, 255, 256, 290])
def test_shared_lengths(mit2, ctx, dtype, shared):
    b = Batch([1, 1, 1], [shared + 1, shared + 40, shared + 3], page=16, dim=64, dtype=dtype, seed=shared)
    _check(mit2, ctx, b, [0, 3], [shared])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [1, 2, 8, 32, 128, 1024])
@pytest.mark.parametrize("alias", [False, True])
def test_pages(mit2, ctx, dtype, page, alias):
    b = Batch([1, 3, 0, 20], [190, 131, 150, 157], page=page, dim=64, dtype=dtype, seed=page, lead_rows=1, tail_rows=2)
    _check(mit2, ctx, b, [0, 4], [130], alias=alias)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new", [(64, (4, 2), [14, 3, 20]), (128, (4, 2), [30, 29, 1]), (64, (2, 2), [100, 81, 0]), (128, (8, 2), [65, 40, 90]),
                                           (256, (2, 1), [70, 5, 6]), (96, (6, 2), [40, 3, 17])])
@pytest.mark.parametrize("tree", [False, True])
def test_many_rows(mit2, ctx, dtype, dim, heads, new, tree):
    b = Batch(new, [n + 300 + 40 * s for s, n in enumerate(new)], page=32, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim, lead_rows=3,
              tail_rows=1)
    context_ref.share(b, [0, 3], [290], True)
    _check(mit2, ctx, b, [0, 3], [290], mask=ops_ref.trees(b, dim)[0] if tree else None, made=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,heads,seqs,shared", [(128, (8, 2), 40, 700), (64, (20, 20), 8, 650), (64, (2, 1), 130, 300), (64, (4, 4), 3, 3000)])
def test_long_prefixes_and_large_groups(mit2, ctx, dtype, dim, heads, seqs, shared):
    lens = [shared + 1 + (13 * s) % 50 for s in range(seqs)]
    b = Batch([1] * seqs, lens, page=64, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=seqs)
    _check(mit2, ctx, b, [0, seqs], [shared])


def test_many_groups(mit2, ctx):
    """More groups, and sequences, than a wave's lanes; empty ones, and sequences outside all groups."""
    seqs = 150
    new = [s % 3 for s in range(seqs)]
    lens = [n + 70 + (11 * s) % 30 for s, n in enumerate(new)]
    b = Batch(new, lens, page=8, kv_heads=1, q_heads=2, dim=32, dtype="f16", seed=9, tail_rows=5, lead_rows=2)
    bounds = [3, 3] + sorted((7 * g) % 140 + 4 for g in range(80)) + [147]
    shared = [(64, 70, 65, 0)[g % 4] for g in range(len(bounds) - 1)]
    _check(mit2, ctx, b, bounds, shared)


def test_no_groups_and_groups_of_one(mit2, ctx):
    b = Batch([1, 5, 1], [200, 90, 700], page=16, dim=64, dtype="bf16", seed=5)
    _check(mit2, ctx, b, [], [])
    _check(mit2, ctx, b, [0, 1, 2, 3], [199, 80, 640])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_more_said_than_there_is(mit2, ctx, dtype):
    """New rows are not shared, whatever is said; nor rows past the shortest sequence's."""
    b = Batch([1, 1, 70], [150, 300, 210], page=16, dim=64, dtype=dtype, seed=6)
    context_ref.share(b, [0, 3], [140], True)
    for said in (141, 150, 1 << 20, 2 ** 31 - 1):
        _check(mit2, ctx, b, [0, 3], [said], made=True, hint=150)
    _check(mit2, ctx, b, [0, 3], [-5], made=True)
    b = Batch([1, 4, 1], [150, 2, 300], page=16, dim=64, dtype=dtype, seed=7)  # one with fewer rows than new ones
    _check(mit2, ctx, b, [0, 3], [140], made=True)
    b = Batch([1, 0, 1], [150, 10, 151], page=16, dim=64, dtype=dtype, seed=7)  # one without new rows is not asked
    for j in range(140):
        for x in (b.k, b.v):
            x[b.page_of(2, j), :, j % 16] = x[b.page_of(0, j), :, j % 16]
    _check(mit2, ctx, b, [0, 3], [140], made=True)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_missing_pages(mit2, ctx, dtype):
    b = Batch([1, 20, 5], [200, 277, 240], page=16, dim=64, dtype=dtype, seed=10)
    context_ref.share(b, [0, 3], [192], True)
    b.table[:, 0] = b.table[:, 3] = -1  # (of the shared rows: for all)
    b.table[1, 13], b.table[2, 14], b.table[1, 16] = b.pages, 2 ** 31 - 1, -2 ** 31
    _check(mit2, ctx, b, [0, 3], [192], made=True)
    b.table[:] = -1
    got = _check(mit2, ctx, b, [0, 3], [192], made=True)
    assert bool((got == 0).all())
    b = Batch([1, 1], [200, 200], page=16, dim=64, dtype=dtype, seed=11)
    context_ref.share(b, [0, 2], [192], True)
    b.length = [b.table.shape[1] * 16 + 9, 200]  # past the table
    _check(mit2, ctx, b, [0, 2], [192], made=True)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_that_see_nothing(mit2, ctx, dtype):
    b = Batch([9, 20, 3], [9, 20, 40], page=16, dim=64, dtype=dtype, seed=7)
    mask = ops_ref.trees(b, 3)[0]
    mask[[0, 4, 8, 9, 28]] = 0
    x = Shared(mit2, b, [0, 3], [64], mask=mask)
    got = x.run(ctx)
    assert bool((got[[0, 4, 8, 9, 28]] == 0).all()) and bool((x.lse[[0, 4, 8, 9, 28]] == -math.inf).all())
    _check(mit2, ctx, b, [0, 3], [64], mask=mask, made=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_large_equal_and_light_scores(mit2, ctx, dtype, new):
    b = Batch([new, 1], [300, 290], dim=64, dtype=dtype, seed=11)
    context_ref.share(b, [0, 2], [250], True)
    b.q *= 8
    b.k *= 4
    for scale in (1.0, 0.0, -0.25):
        _check(mit2, ctx, b, [0, 2], [250], scale=scale, made=True, what=f"{dtype} scale {scale}")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_heavy_keys_on_one_side(mit2, ctx, dtype):
    """One key has all the weight: among the shared rows, or among a sequence's own; the other side's part counts for nothing."""
    for heavy in (10, 250):
        b = Batch([1, 3], [300, 280], dim=64, dtype=dtype, seed=12)
        context_ref.share(b, [0, 2], [200], True)
        b.q[..., 0] = 60.0
        for s in range(2):
            b.k[b.page_of(s, heavy), :, heavy % b.page, 0] = 60.0
        _check(mit2, ctx, b, [0, 2], [200], scale=1.0, made=True, what=f"{dtype} heavy {heavy}")


def test_what_is_not_finite_is_not_seen(mit2, ctx):
    b = Batch([1, 6], [150, 160], page=16, dim=64, dtype="bf16", seed=8)
    context_ref.share(b, [0, 2], [140], True)
    clean = Shared(mit2, b, [0, 2], [140]).run(ctx)
    used = np.zeros((b.pages, b.page), bool)
    for s, n in enumerate(b.length):
        for j in range(n):
            used[b.page_of(s, j), j % b.page] = True
    for cache in (b.k, b.v):
        cache.permute(0, 2, 1, 3)[torch.from_numpy(~used)] = math.nan
    assert torch.equal(Shared(mit2, b, [0, 2], [140]).run(ctx), clean)
    b.v[b.page_of(1, 159), :, 159 % 16, 5] = math.inf  # the last new row of the second: seen by itself
    got = Shared(mit2, b, [0, 2], [140]).run(ctx)
    assert torch.equal(got[:-1], clean[:-1]) and bool((got[-1, :, 5] == math.inf).all())


def test_strides(mit2, ctx):
    """Queries in a projection's rows at an odd stride, outputs head by head."""
    b = Batch([1, 12, 33], [160, 170, 200], q_heads=4, kv_heads=2, dim=64, dtype="f16", seed=12)
    context_ref.share(b, [0, 3], [150], True)
    ref = Shared(mit2, b, [0, 3], [150]).run(ctx)
    x = Shared(mit2, b, [0, 3], [150])
    width = b.q_heads * b.dim + 5
    q = torch.zeros(b.rows * width + 1, dtype=TORCH["f16"], device=DEV)
    q[1:].view(b.rows, width)[:, : b.q_heads * b.dim] = x.on.q.reshape(b.rows, -1)
    out = torch.full((b.q_heads, b.rows, b.dim), math.nan, dtype=TORCH["f16"], device=DEV)
    x.args.q, x.args.q_row = q.data_ptr() + 2, width
    x.args.out, x.args.out_row, x.args.out_head = out.data_ptr(), b.dim, b.rows * b.dim
    x.run(ctx)
    assert torch.equal(out.permute(1, 0, 2).double().cpu(), ref)


@pytest.mark.parametrize("new", [1, 40])
def test_any_hints_the_same_bits_again_and_no_lse(mit2, ctx, new):
    b = Batch([new, 1, 2], [900, 970, 880], dim=64, dtype="f32", seed=13)
    context_ref.share(b, [0, 3], [800], True)
    ref, tol = ops_ref.attention64(b, 0.125)
    for rows_hint, hint in ((0, 0), (1, 1000), (970, 1), (1 << 20, 800), (2 ** 32 - 1, 2 ** 32 - 1), (970, 800)):
        x = Shared(mit2, b, [0, 3], [800], hint=hint, lse=False)
        x.on.rows.max_length = rows_hint
        got = x.run(ctx)
        check(got, ref, tol, f"hints {rows_hint} {hint}")
        assert torch.equal(x.run(ctx), got) and bool(torch.isnan(x.lse).all())


@pytest.mark.parametrize("seqs", [0, 2])
def test_nothing_to_do(mit2, ctx, seqs):
    b = Batch([1, 1], [4, 4], dim=64, dtype="f32", seed=15)
    x = Shared(mit2, b, [0, 2], [3])
    x.on.rows.seqs, x.on.rows.rows = seqs, 0 if seqs else 2
    assert bool(torch.isnan(x.run(ctx)).all())


def test_offsets_past_32_bits(mit2, ctx):
    pages, heads, page, dim = 70000, 8, 64, 128
    b = Batch([1, 5], [200, 240], page=page, kv_heads=heads, q_heads=heads, dim=dim, dtype="bf16", seed=16)
    context_ref.share(b, [0, 2], [192], True)
    x = Shared(mit2, b, [0, 2], [192])
    big = [torch.empty(pages * heads * page * dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    try:
        shift = pages - b.pages
        for flat, small in zip(big, (x.on.k, x.on.v)):
            flat.view(pages, heads, page, dim)[shift:] = small
        x.on.table += shift * (x.on.table >= 0)
        x.on.cache.k, x.on.cache.v, x.on.cache.pages = big[0].data_ptr(), big[1].data_ptr(), pages
        ref, tol = ops_ref.attention64(b, dim ** -0.5)
        check(x.run(ctx), ref, tol, "far pages")
    finally:
        del big, x
        torch.cuda.empty_cache()
