"""The paged-cache operators (mit2cfm_kv_append_device, mit2cfm_kv_attention_device) on the GPU against plain 64-bit
restatements (ops_ref.py), where they can go wrong: lengths around tiles and pages, rows that see nothing, unseen NaN
and infinities, entries that are no page, strides, rows of no sequence, offsets past 32 bits, graphs."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ops_ref  # noqa: E402
from ops_ref import HALF_STEP, TORCH, U, Batch  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx(mit2):
    c = mit2.Context(synthetic_seed=3, device=0)
    yield c
    c.close()


class On:
    """A batch's buffers on the GPU and the library's descriptions of them."""

    def __init__(self, mit2, b: Batch):
        self.mit2, self.b = mit2, b
        self.k, self.v, self.q = b.k.to(DEV), b.v.to(DEV), b.q.to(DEV)
        self.new_k, self.new_v = b.new_k.to(DEV), b.new_v.to(DEV)
        self.table, self.start = torch.from_numpy(b.table).to(DEV), torch.from_numpy(b.start).to(DEV)
        self.length = torch.tensor(b.length, dtype=torch.int32, device=DEV)
        self.out = torch.full(b.q.shape, math.nan, dtype=TORCH[b.dtype], device=DEV)
        self.cache = mit2.KvCache(k=self.k.data_ptr(), v=self.v.data_ptr(), table=self.table.data_ptr(), pages=b.pages, page_rows=b.page,
                                  kv_heads=b.kv_heads, head_dim=b.dim, table_stride=b.table.shape[1], dtype=mit2.DTYPES[b.dtype])
        self.rows = mit2.KvRows(start=self.start.data_ptr(), length=self.length.data_ptr(), seqs=len(b.new), rows=b.rows,
                                max_length=max(b.length + [0]))

    def append_args(self, position=None, rot=0, interleaved=False, theta=10000.0):
        b, d = self.b, self.b.dim
        self.position = None if position is None else torch.as_tensor(position, dtype=torch.int32, device=DEV)
        return self.mit2.KvAppend(k=self.new_k.data_ptr(), v=self.new_v.data_ptr(), k_row=b.kv_heads * d, k_head=d, v_row=b.kv_heads * d, v_head=d,
                                  q=self.q.data_ptr(), q_out=self.out.data_ptr(), q_row=b.q_heads * d, q_head=d, q_out_row=b.q_heads * d, q_out_head=d,
                                  q_heads=b.q_heads, position=None if position is None else self.position.data_ptr(), rotary_dim=rot,
                                  interleaved=int(interleaved), theta=theta)

    def attention_args(self, scale=None, mask=None):
        b, d = self.b, self.b.dim
        n = self.mit2.kv_attention_workspace(self.cache, self.rows, b.q_heads)
        self.workspace = torch.full((n + 256,), 255, dtype=torch.uint8, device=DEV)  # (NaN, were it read before it is written)
        self.mask = None if mask is None else torch.from_numpy(mask.view(np.int32)).to(DEV)
        return self.mit2.KvAttention(q=self.q.data_ptr(), out=self.out.data_ptr(), q_row=b.q_heads * d, q_head=d, out_row=b.q_heads * d, out_head=d,
                                     q_heads=b.q_heads, scale=d ** -0.5 if scale is None else scale,
                                     mask=None if mask is None else self.mask.data_ptr(), mask_words=0 if mask is None else mask.shape[1],
                                     workspace=self.workspace.data_ptr(), workspace_bytes=n)

    def attend(self, ctx, **kw):
        a = self.attention_args(**kw)
        torch.cuda.synchronize()
        ctx.kv_attention_device(self.cache, self.rows, a, sync=True)
        assert bool((self.workspace[a.workspace_bytes:] == 255).all())
        return self.out.double().cpu()


def _mine(b):
    """Whether a row is a sequence's."""
    m = torch.zeros(b.rows, dtype=torch.bool)
    m[int(b.start[0]): int(b.start[-1])] = True
    return m


def _check(got, ref, tol, what):
    off = (got - ref).abs()
    off[torch.isnan(got) & torch.isnan(ref)] = 0.0
    off = torch.nan_to_num(off, nan=math.inf)
    worst = float((off / tol.clamp_min(1e-300)).amax()) if off.numel() else 0.0
    print(f"{what}: worst {worst:.3f} of the tolerance", flush=True)
    assert bool((off <= tol).all()), what


def _check_attention(ctx, mit2, b, mask=None, scale=None, what=""):
    on = On(mit2, b)
    got = on.attend(ctx, mask=mask, scale=scale)
    ref, tol = ops_ref.attention64(b, b.dim ** -0.5 if scale is None else scale, mask)
    mine = _mine(b)
    assert bool(torch.isnan(got[~mine]).all()), "rows of no sequence were written"
    _check(got[mine], ref[mine], tol[mine], what or f"{b.dtype} dim {b.dim} page {b.page} heads {b.q_heads}/{b.kv_heads}")
    return got


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 0, False), (64, 64, True), (64, 64, False), (128, 96, False), (96, 32, True), (32, 10, False),
                                                 (32, 6, True), (256, 256, False), (192, 48, False)])
def test_append_rotates_and_places(mit2, ctx, dtype, dim, rot, interleaved):
    b = Batch([1, 0, 5, 17, 2], [1, 0, 5, 40, 130], page=16, kv_heads=2, q_heads=6, dim=dim, dtype=dtype, seed=dim + rot, tail_rows=3, lead_rows=2)
    _append_check(mit2, ctx, b, rot, interleaved)


@pytest.mark.parametrize("page", [1, 8, 64, 1024])
def test_append_pages(mit2, ctx, page):
    _append_check(mit2, ctx, Batch([3, 9], [3, 70], page=page, dim=64, dtype="f16", seed=page), 64, False)


def test_append_many_rows_and_sequences(mit2, ctx):
    """Rows enough that blocks take several, sequences more than a wave's lanes, some without rows."""
    new = [(7 * s) % 31 for s in range(150)]
    _append_check(mit2, ctx, Batch(new, [n + (11 * s) % 50 for s, n in enumerate(new)], page=8, kv_heads=1, q_heads=2, dim=64, dtype="bf16", seed=9,
                                   tail_rows=5), 64, True)


@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_append_far_and_negative_positions(mit2, ctx, theta):
    """Angles of far positions keep fp32's precision."""
    b = Batch([6], [9], dim=64, dtype="f32", seed=2)
    _append_check(mit2, ctx, b, 64, False, position=np.array([0, -3, 131071, 1000003, 16777217, 2147483647], np.int32), theta=theta)


def _append_check(mit2, ctx, b, rot, interleaved, position=None, theta=10000.0):
    on = On(mit2, b)
    a = on.append_args(position=position, rot=rot, interleaved=interleaved, theta=theta)
    torch.cuda.synchronize()
    ctx.kv_append_device(on.cache, on.rows, a, sync=True)
    q, k, v = ops_ref.append64(b, position, rot, interleaved, theta)
    # a turned element is two products and their sum, with a cosine and a sine that are each off by the angle's rounding to fp32
    # in half turns (pi 2^-24), a few ulp of their own, and far out by the fp64 product's 2^-52 of the turns; then the type's rounding
    turns = 0.16 * max([abs(int(p)) for p in (position if position is not None else b.length)] + [1]) * 2.0 ** -52 * 2 * math.pi * 4
    size = torch.maximum(b.q.double().abs().amax(-1, keepdim=True), b.new_k.double().abs().max())
    e = 2 * size * (math.pi * U + 6 * U + turns)
    _check(on.out.double().cpu(), q, torch.where(torch.isnan(q), 0.0, e + HALF_STEP[b.dtype] * (q.abs() + e)), f"q {b.dtype} {b.dim}/{rot}")
    e = 2 * float(b.new_k.double().abs().max()) * (math.pi * U + 6 * U + turns)
    changed = k != b.k.double()
    _check(on.k.double().cpu(), k, torch.where(changed, e + HALF_STEP[b.dtype] * (k.abs() + e), 0.0), f"k {b.dtype} {b.dim}/{rot}")
    assert torch.equal(on.v.double().cpu(), v)


def test_append_rows_without_a_page_are_dropped(mit2, ctx):
    b = Batch([4, 4, 3], [20, 36, 3], page=16, dim=64, dtype="f32", seed=4)
    b.table[0, 1], b.table[1, 2], b.table[2, 0] = -1, b.pages, 2 ** 31 - 1
    _append_check(mit2, ctx, b, 0, False)
    b = Batch([2, 3], [2, 3], page=16, dim=64, dtype="f32", seed=5)
    b.length = [1, 100]  # before the sequence's begin; past its table
    _append_check(mit2, ctx, b, 64, False)


def test_append_strides_in_place_and_without_queries(mit2, ctx):
    """q, k and v as slices of one projection's rows (an odd row stride: element-wise), q rotated in place; then no q."""
    b = Batch([3, 6], [3, 30], page=8, kv_heads=2, q_heads=4, dim=64, dtype="f16", seed=6)
    for pad in (8, 3):
        on = On(mit2, b)
        width = (b.q_heads + 2 * b.kv_heads) * b.dim + pad
        packed = torch.zeros(b.rows, width, dtype=TORCH[b.dtype], device=DEV)
        packed[:, : b.q_heads * b.dim] = on.q.reshape(b.rows, -1)
        packed[:, b.q_heads * b.dim: (b.q_heads + b.kv_heads) * b.dim] = on.new_k.reshape(b.rows, -1)
        packed[:, (b.q_heads + b.kv_heads) * b.dim: (b.q_heads + 2 * b.kv_heads) * b.dim] = on.new_v.reshape(b.rows, -1)
        a = on.append_args(rot=64, interleaved=True)
        at = packed.data_ptr()
        a.q = a.q_out = at
        a.k, a.v = at + 2 * b.q_heads * b.dim, at + 2 * (b.q_heads + b.kv_heads) * b.dim
        a.q_row = a.k_row = a.v_row = a.q_out_row = width
        torch.cuda.synchronize()
        ctx.kv_append_device(on.cache, on.rows, a, sync=True)
        plain = On(mit2, b)
        ctx.kv_append_device(plain.cache, plain.rows, plain.append_args(rot=64, interleaved=True), sync=True)
        assert torch.equal(packed[:, : b.q_heads * b.dim].reshape(plain.out.shape), plain.out)
        assert torch.equal(on.k, plain.k) and torch.equal(on.v, plain.v)
        a = on.append_args(rot=64, interleaved=True)
        a.q, a.q_out, a.q_heads = None, None, 0
        on.k.copy_(b.k)
        torch.cuda.synchronize()
        ctx.kv_append_device(on.cache, on.rows, a, sync=True)
        assert torch.equal(on.k, plain.k)


# ------------------------------------------------------------------ attention
LENGTHS = [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,q_heads,kv_heads", [(64, 20, 20), (64, 8, 8), (128, 8, 2), (32, 7, 1), (96, 6, 1), (192, 4, 2), (256, 3, 1),
                                                  (128, 16, 1), (64, 34, 2), (32, 70, 1)])
def test_attention_of_single_tokens(mit2, ctx, dtype, dim, q_heads, kv_heads):
    b = Batch([1] * len(LENGTHS), LENGTHS, page=16, kv_heads=kv_heads, q_heads=q_heads, dim=dim, dtype=dtype, seed=dim)
    _check_attention(ctx, mit2, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [1, 2, 8, 32, 128, 1024])
def test_attention_pages(mit2, ctx, dtype, page):
    _check_attention(ctx, mit2, Batch([1, 3, 0, 20], [90, 131, 0, 57], page=page, dim=64, dtype=dtype, seed=page, lead_rows=1, tail_rows=2))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,length", [([1], [3001]), ([1, 1], [5000, 3]), ([2], [2600]), ([70], [1200]), ([17, 40], [700, 40]), ([1] * 5, [999] * 5)])
def test_attention_of_long_caches(mit2, ctx, dtype, new, length):
    _check_attention(ctx, mit2, Batch(new, length, page=64, kv_heads=1, q_heads=2, dim=64, dtype=dtype, seed=sum(new)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads", [(64, (4, 4)), (128, (8, 2)), (96, (5, 1))])
def test_attention_of_trees(mit2, ctx, dtype, dim, heads):
    b = Batch([33, 1, 0, 64, 7, 90], [33, 50, 9, 300, 7, 91], page=16, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim, tail_rows=2)
    _check_attention(ctx, mit2, b, mask=ops_ref.trees(b, dim)[0])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [1, 4, 8, 16, 64, 256])
@pytest.mark.parametrize("dim,heads,new", [(64, (4, 2), [14]), (128, (4, 2), [30, 29]), (64, (2, 2), [100, 81]), (128, (8, 2), [65, 40, 90]),
                                           (256, (2, 1), [70])])
def test_attention_of_many_rows_over_pages(mit2, ctx, dtype, page, dim, heads, new):
    """Each form of the tiles (28, 60, 90 and 260 query rows on average, large heads), pages smaller and larger than a tile."""
    b = Batch(new, [n + (130, 7, 300)[s] for s, n in enumerate(new)], page=page, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype,
              seed=page + dim, lead_rows=3, tail_rows=1)
    _check_attention(ctx, mit2, b)
    _check_attention(ctx, mit2, b, mask=ops_ref.trees(b, page)[0])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_many_rows_with_missing_pages_and_splits(mit2, ctx, dtype, dim):
    b = Batch([150, 3, 200], [2900, 3, 1500], page=32, q_heads=2, kv_heads=1, dim=dim, dtype=dtype, seed=dim)
    b.table[0, 5], b.table[0, 60], b.table[2, 0], b.table[2, 46] = -1, b.pages, -7, 2 ** 31 - 1
    _check_attention(ctx, mit2, b)
    _check_attention(ctx, mit2, b, mask=ops_ref.trees(b, 1)[0])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,tree", [(64, (2, 2), True), (128, (8, 2), True), (64, (2, 2), False), (128, (4, 1), False), (96, (4, 1), False)])
def test_many_rows_are_blind_to_what_they_do_not_see(mit2, ctx, dtype, dim, heads, tree):
    """The same for tiles of many rows: NaN and infinities among the new rows and behind the sequences' ends."""
    b = Batch([100, 70], [230, 75], page=16, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=22)
    mask = ops_ref.trees(b, 9)[0] if tree else None
    clean = On(mit2, b).attend(ctx, mask=mask)
    used = np.zeros((b.pages, b.page), bool)
    for s, n in enumerate(b.length):
        for j in range(n):
            used[b.page_of(s, j), j % b.page] = True
    for cache in (b.k, b.v):
        cache.permute(0, 2, 1, 3)[torch.from_numpy(~used)] = math.nan
    assert torch.equal(On(mit2, b).attend(ctx, mask=mask), clean)
    sees = torch.zeros(b.rows, 2, dtype=torch.bool)  # row sees the NaN, the infinity
    for which, (s, i, value) in enumerate(((0, 61, math.nan), (1, 20, -math.inf))):
        j = b.length[s] - b.new[s] + i
        b.v[b.page_of(s, j), :, j % b.page, 5] = value
        for row, s2, i2, _ in b.each_row():
            sees[row, which] = s2 == s and bool(i2 >= i if mask is None else mask[row, i // 32] >> np.uint32(i % 32) & 1)
    got = On(mit2, b).attend(ctx, mask=mask)
    hit = sees.any(1)
    assert torch.equal(got[~hit], clean[~hit])
    assert bool(torch.isnan(got[sees[:, 0]][:, :, 5]).all()) and bool((got[sees[:, 1]][:, :, 5] == -math.inf).all())
    rest = [d for d in range(dim) if d != 5]
    assert torch.equal(got[hit][:, :, rest], clean[hit][:, :, rest])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_a_mask_of_too_few_words(mit2, ctx, dtype):
    """New rows past the mask's words are seen by none."""
    b = Batch([40], [60], dim=64, dtype=dtype, seed=1)
    _check_attention(ctx, mit2, b, mask=np.full((40, 1), 0xFFFFFFFF, np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_rows_that_see_nothing_give_zero(mit2, ctx, dtype):
    b = Batch([9, 20, 3], [9, 20, 40], page=16, dim=64, dtype=dtype, seed=7)
    mask = ops_ref.trees(b, 3)[0]
    mask[[0, 4, 8, 9, 28]] = 0
    got = _check_attention(ctx, mit2, b, mask=mask)
    assert bool((got[[0, 4, 8, 9, 28]] == 0).all())
    b.table[1:] = -1  # no pages at all
    got = _check_attention(ctx, mit2, b, mask=mask)
    assert bool((got[9:] == 0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_is_blind_to_what_a_row_does_not_see(mit2, ctx, dtype):
    """NaN and infinities in spare pages, behind a sequence's end and in new rows that a row does not see leave it as it was; a
    row that sees them has them."""
    b = Batch([6, 40, 1], [21, 55, 3], page=16, dim=64, dtype=dtype, seed=8)
    mask = ops_ref.trees(b, 5)[0]
    clean = On(mit2, b).attend(ctx, mask=mask)
    used = np.zeros((b.pages, b.page), bool)
    for s, n in enumerate(b.length):
        for j in range(n):
            used[b.page_of(s, j), j % b.page] = True
    dirty = torch.from_numpy(~used)
    for cache, value in ((b.k, math.nan), (b.v, math.inf)):
        cache.permute(0, 2, 1, 3)[dirty] = value
    assert torch.equal(On(mit2, b).attend(ctx, mask=mask), clean)
    # new row 3 of sequence 0 and 30 of sequence 1: seen by themselves and by their children alone
    hit = torch.zeros(b.rows, dtype=torch.bool)
    for s, i, value in ((0, 3, math.nan), (1, 30, math.inf)):
        j = b.length[s] - b.new[s] + i
        b.v[b.page_of(s, j), :, j % b.page, 5] = value
        b.k[b.page_of(s, j), :, j % b.page, 7] = math.nan if s == 0 else b.k[b.page_of(s, j), :, j % b.page, 7]
        for row, s2, _, _ in b.each_row():
            hit[row] |= s2 == s and bool(mask[row, i // 32] >> np.uint32(i % 32) & 1)
    got = On(mit2, b).attend(ctx, mask=mask)
    assert torch.equal(got[~hit], clean[~hit])
    assert not bool(torch.isfinite(got[hit][:, :, 5]).any())
    inf = hit.clone()
    inf[: b.start[1]] = False
    assert bool((got[inf][:, :, 5] == math.inf).all()) and bool(torch.isfinite(got[inf][:, :, :5]).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_entries_that_are_no_page_are_unseen(mit2, ctx, dtype):
    b = Batch([1, 20, 5], [100, 77, 40], page=16, dim=64, dtype=dtype, seed=10)
    b.table[0, 0], b.table[0, 3], b.table[1, 4], b.table[2, 1] = -1, b.pages, 2 ** 31 - 1, -2 ** 31
    _check_attention(ctx, mit2, b)
    b.length = [b.table.shape[1] * 16 + 9, 77, 3]  # past the table: what the table holds; fewer rows than new ones
    _check_attention(ctx, mit2, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_of_large_and_equal_scores(mit2, ctx, dtype):
    """Scores in the hundreds, alike for all keys or far apart."""
    b = Batch([1, 4], [300, 90], dim=64, dtype=dtype, seed=11)
    b.q *= 8
    b.k *= 4
    _check_attention(ctx, mit2, b, scale=1.0)
    _check_attention(ctx, mit2, b, scale=0.0)
    _check_attention(ctx, mit2, b, scale=-0.25)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 20, 130])
@pytest.mark.parametrize("light", [13.4, 17.9])
def test_attention_of_many_light_keys(mit2, ctx, dtype, new, light):
    """One heavy key in 32, with values of 0, beside keys whose weights are e^-light of it: what they add up to is all there is."""
    b = Batch([new], [1500], dim=64, dtype=dtype, seed=31)
    b.q.zero_()
    b.q[..., 0] = 1.0
    for j in range(1500):
        page, slot = b.page_of(0, j), j % b.page
        b.k[page, :, slot, 0] = 0.0 if j % 32 == 0 else -light
        b.v[page, :, slot] = 0.0 if j % 32 == 0 else b.v[page, :, slot].abs() * 16 + 16
    on = On(mit2, b)
    got = on.attend(ctx, scale=1.0)
    ref, tol = ops_ref.attention64(b, 1.0)
    if dtype == "f16":
        # weights are taken at 2^7 times their size: below the type's smallest normal each is off by at most half its step, 2^-25, of that; 31
        # of them to a weight of 1.  A result below the smallest normal is rounded by as much.
        tol = tol + 31 * 2.0 ** -32 * float(b.v.abs().max()) + 2.0 ** -25
    _check(got[_mine(b)], ref[_mine(b)], tol[_mine(b)], f"light keys {dtype} {new} {light}")


def test_attention_strides(mit2, ctx):
    """Queries in a projection's rows at an odd stride, outputs head by head."""
    b = Batch([1, 12, 33], [60, 70, 200], q_heads=4, kv_heads=2, dim=64, dtype="f16", seed=12)
    for dtype in ("f16", "f32"):
        b.dtype = dtype
        for name in ("k", "v", "q", "new_k", "new_v"):
            setattr(b, name, getattr(b, name).to(TORCH[dtype]))
        ref = On(mit2, b).attend(ctx)
        on = On(mit2, b)
        width = b.q_heads * b.dim + 5
        q = torch.zeros(b.rows * width + 1, dtype=TORCH[dtype], device=DEV)
        q[1:].view(b.rows, width)[:, : b.q_heads * b.dim] = on.q.reshape(b.rows, -1)
        out = torch.full((b.q_heads, b.rows, b.dim), math.nan, dtype=TORCH[dtype], device=DEV)
        a = on.attention_args()
        a.q, a.q_row = q.data_ptr() + q.element_size(), width
        a.out, a.out_row, a.out_head = out.data_ptr(), b.dim, b.rows * b.dim
        torch.cuda.synchronize()
        ctx.kv_attention_device(on.cache, on.rows, a, sync=True)
        assert torch.equal(out.permute(1, 0, 2).double().cpu(), ref)


def test_attention_does_not_depend_on_the_length_hint_or_the_batch_beyond_rounding(mit2, ctx):
    b = Batch([1, 1, 5], [2000, 70, 400], dim=64, dtype="f32", seed=13)
    ref, tol = ops_ref.attention64(b, 0.125)
    for hint in (0, 1, 100, 1 << 20, 2 ** 32 - 1):
        on = On(mit2, b)
        on.rows.max_length = hint
        _check(on.attend(ctx), ref, tol, f"hint {hint}")


def test_the_same_call_gives_the_same_bits(mit2, ctx):
    b = Batch([1, 30, 1], [2600, 900, 5], dim=128, dtype="bf16", seed=14)
    on = On(mit2, b)
    first = on.attend(ctx)
    for _ in range(3):
        assert torch.equal(on.attend(ctx), first)


@pytest.mark.parametrize("seqs", [0, 2])
def test_nothing_to_do(mit2, ctx, seqs):
    b = Batch([1, 1], [4, 4], dim=64, dtype="f32", seed=15)
    on = On(mit2, b)
    on.rows.seqs, on.rows.rows = seqs, 0 if seqs else 2
    assert bool(torch.isnan(on.attend(ctx)).all())
    ctx.kv_append_device(on.cache, on.rows, on.append_args(), sync=True)
    assert torch.equal(on.k.cpu(), b.k) and bool(torch.isnan(on.out).all())


def test_offsets_past_32_bits(mit2, ctx):
    """A cache of over 2^32 elements: rows appended to its last pages and read there."""
    pages, heads, page, dim = 70000, 8, 64, 128
    b = Batch([1, 5], [100, 40], page=page, kv_heads=heads, q_heads=heads, dim=dim, dtype="bf16", seed=16)
    on = On(mit2, b)
    n = pages * heads * page * dim
    big = [torch.empty(n, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    try:
        shift = pages - b.pages
        for flat, small in zip(big, (on.k, on.v)):
            flat.view(pages, heads, page, dim)[shift:] = small
        on.table += shift * (on.table >= 0)
        on.cache.k, on.cache.v, on.cache.pages = big[0].data_ptr(), big[1].data_ptr(), pages
        a = on.append_args(rot=128)
        torch.cuda.synchronize()
        ctx.kv_append_device(on.cache, on.rows, a, sync=True)
        _, k, v = ops_ref.append64(b, None, 128, False, 10000.0)
        got = big[0].view(pages, heads, page, dim)[shift:].cpu()
        assert float((got.double() - k).abs().max()) <= 2.0 ** -8 * float(k.abs().max())
        b.k, b.v = got, v.to(torch.bfloat16)
        ref, tol = ops_ref.attention64(b, dim ** -0.5)
        _check(on.attend(ctx), ref, tol, "far pages")
    finally:
        del big, on
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new", [(64, (20, 20), [25, 1, 9]), (128, (32, 8), [63, 40, 0, 12]), (96, (6, 2), [40, 3])])
def test_drafted_trees_appended_and_attended(mit2, ctx, dtype, dim, heads, new):
    """A draft's check as it is used: the trees' rows appended at their depths' positions, their queries rotated on the way, and
    attended over the cache, one call behind the other."""
    b = Batch(new, [n + 70 * (s + 1) for s, n in enumerate(new)], page=16, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim, tail_rows=1)
    mask, depth = ops_ref.trees(b, 21)
    position = np.zeros(b.rows, np.int32)
    for row, s, _, before in b.each_row():
        position[row] = before + depth[row]
    on = On(mit2, b)
    put, att = on.append_args(position=position, rot=dim), on.attention_args(mask=mask)
    out = torch.full_like(on.out, math.nan)
    att.q, att.out = on.out.data_ptr(), out.data_ptr()
    torch.cuda.synchronize()
    ctx.kv_append_device(on.cache, on.rows, put)
    ctx.kv_attention_device(on.cache, on.rows, att, sync=True)
    q, k, v = ops_ref.append64(b, position, dim, False, 10000.0)
    for got, want, step in ((on.out, q, 1.0), (on.k, k, 1.0), (on.v, v, 0.0)):
        off = (got.double().cpu() - want).abs().nan_to_num(0.0)
        assert bool((off <= step * (HALF_STEP[dtype] * want.abs().nan_to_num(0.0) + 2e-6 * 8)).all())
    b.q, b.k, b.v = on.out.cpu(), on.k.cpu(), on.v.cpu()  # (what the attention was given)
    ref, tol = ops_ref.attention64(b, dim ** -0.5, mask)
    mine = _mine(b)
    _check(out.double().cpu()[mine], ref[mine], tol[mine], f"trees {dtype} {dim}")


class Graph:
    """The context's stream captured into a graph."""

    def __init__(self, ctx, enqueue):
        self.hip, self.stream = ctypes.CDLL("libamdhip64.so.7"), ctypes.c_void_p(ctx.stream)
        self.graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0  # hipStreamCaptureModeThreadLocal
        try:
            enqueue()
        finally:
            assert self.hip.hipStreamEndCapture(self.stream, ctypes.byref(self.graph)) == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exe), self.graph, None, None, ctypes.c_size_t(0)) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exe, self.stream) == 0
        assert self.hip.hipStreamSynchronize(self.stream) == 0

    def close(self):
        self.hip.hipGraphExecDestroy(self.exe)
        self.hip.hipGraphDestroy(self.graph)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_graph_replays_follow_lengths_on_the_device(mit2, ctx, dtype):
    """Append and attention captured once; every replay, with the sequences grown in between and eager calls before it, equals the
    eager calls."""
    b = Batch([1, 1], [700, 90], page=16, dim=64, dtype=dtype, seed=17, spare=0, extra_entries=0)
    on, eager = On(mit2, b), On(mit2, b)
    calls = []
    for o in (on, eager):
        calls.append((o.append_args(rot=64), o.attention_args()))
    torch.cuda.synchronize()

    def enqueue(o, c):
        ctx.kv_append_device(o.cache, o.rows, c[0])
        ap, at = c
        at.q, at.out = ap.q, ap.q_out
        ctx.kv_attention_device(o.cache, o.rows, at)

    g = Graph(ctx, lambda: enqueue(on, calls[0]))
    try:
        for lens in ([640, 3], [650, 4], [651, 5], [700, 80]):
            for o in (on, eager):
                o.length.copy_(torch.tensor(lens, dtype=torch.int32))
                o.q.normal_(generator=torch.Generator(device=DEV).manual_seed(lens[0]))
            torch.cuda.synchronize()
            enqueue(eager, calls[1])
            ctx.synchronize()
            g.replay()
            assert torch.equal(on.out, eager.out) and torch.equal(on.k, eager.k), lens
    finally:
        g.close()


def test_two_contexts_at_once(mit2, ctx):
    """Calls of two contexts on their own streams, with a workspace each, give what they give alone."""
    other = mit2.Context(synthetic_seed=3, device=0)
    try:
        sets = [On(mit2, Batch([1] * 4, [2500, 100, 1800, 7], dim=64, dtype="bf16", seed=s)) for s in (18, 19)]
        alone = [o.attend(ctx) for o in sets]
        args = [o.attention_args() for o in sets]
        torch.cuda.synchronize()
        for _ in range(20):
            for c, o, a in zip((ctx, other), sets, args):
                c.kv_attention_device(o.cache, o.rows, a)
        torch.cuda.synchronize()
        for o, ref in zip(sets, alone):
            assert torch.equal(o.out.double().cpu(), ref)
    finally:
        other.close()
