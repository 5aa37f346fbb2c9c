"""Eviction from paged caches (mit2cfm_kv_evict_device) on the GPU against a plain restatement (context_ref.py): whole numbers and
copies, so everything is equal to the bit."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
from context_ref import DEV  # noqa: E402
from ops_ref import TORCH  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(mit2):
    c = mit2.Context(synthetic_seed=3, device=0)
    yield c
    c.close()


class Cut:
    """A call's buffers; what must not be written holds NaN and -1."""

    def __init__(self, mit2, length, keep, *, layers=2, heads=2, dim=32, page=8, dtype="f32", first=2, last=3, stride=None, born=False, in_place=False, seed=0,
                 weights=None, hint=None, spare=2, capacity=None):
        rng = np.random.default_rng(seed)
        seqs = len(length)
        entries = -(-max([1] + list(capacity or length)) // page) + 1
        pages = seqs * entries + spare
        self.table = rng.permutation(pages)[: seqs * entries].reshape(seqs, entries).astype(np.int32)
        self.length, self.keep, self.page, self.first, self.last, self.dtype = list(length), list(keep), page, first, last, dtype
        stride = stride or entries * page
        g = torch.Generator().manual_seed(seed)
        self.k, self.v = (torch.randn(layers, pages, heads, page, dim, generator=g).to(TORCH[dtype]) for _ in range(2))
        self.weights = rng.exponential(1.0, (layers, seqs, heads, stride)).astype(np.float32) if weights is None else weights
        self.born = self.now = None
        if born:
            self.born = rng.permuted(np.broadcast_to(np.arange(stride, dtype=np.int32) * 2 - 5, self.weights.shape), axis=-1)
            self.now = np.array([2 * n - 7 for n in length], np.int32)
        self.in_place, self.hint, self.mit2 = in_place, hint, mit2

    def upload(self):
        mit2 = self.mit2
        layers, seqs, heads, stride = self.weights.shape

        def up(x):
            return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(DEV)

        self.dk, self.dv, self.dt, self.dw, self.db, self.dn = self.k.to(DEV), self.v.to(DEV), up(self.table), up(self.weights), up(self.born), up(self.now)
        self.dl, self.dkeep = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (self.length, self.keep))
        self.out_w = self.dw if self.in_place else torch.full_like(self.dw, float("nan"))
        self.out_b = None if self.db is None else self.db if self.in_place else torch.full_like(self.db, -1)
        self.out_l = self.dl if self.in_place else torch.full_like(self.dl, -9)
        dim = self.k.shape[-1]
        self.cache = mit2.KvCache(k=self.dk.data_ptr(), v=self.dv.data_ptr(), table=self.dt.data_ptr(), pages=self.k.shape[1], page_rows=self.page,
                                  kv_heads=heads, head_dim=dim, table_stride=self.table.shape[1], dtype=mit2.DTYPES[self.dtype])

        def at(x):
            return None if x is None else x.data_ptr()

        self.args = mit2.KvEvict(seqs=seqs, layers=layers, layer_stride=self.dk.stride(0), length=at(self.dl), keep=at(self.dkeep), first_rows=self.first,
                                 last_rows=self.last, max_length=max([0] + self.length) if self.hint is None else self.hint, weights=at(self.dw),
                                 weights_out=at(self.out_w), weight_stride=stride, born=at(self.db), born_out=at(self.out_b), now=at(self.dn),
                                 length_out=at(self.out_l))
        n = mit2.kv_evict_workspace(self.cache, self.args)
        assert n > 0
        self.workspace = torch.full((n + 256,), 255, dtype=torch.uint8, device=DEV)
        self.args.workspace, self.args.workspace_bytes = self.workspace.data_ptr(), n
        torch.cuda.synchronize()

    def expect(self):
        return context_ref.evict(self.k.double().numpy(), self.v.double().numpy(), self.table, self.page, self.length, self.keep, self.weights, self.first,
                                 self.last, self.born, self.now)

    def compare(self):
        k, v, w, b, n = self.expect()
        assert self.out_l.cpu().tolist() == n.tolist()
        assert np.array_equal(self.dk.double().cpu().numpy(), k) and np.array_equal(self.dv.double().cpu().numpy(), v)
        got = self.out_w.cpu().numpy()
        told = np.broadcast_to(np.arange(w.shape[3]) < n[:, None], w.shape[:2] + (w.shape[3],))[:, :, None] & np.ones(w.shape, bool)
        assert np.array_equal(got[told], w[told], equal_nan=True)
        assert np.array_equal(got[~told], self.weights[~told] if self.in_place else w[~told], equal_nan=True)
        if self.born is not None:
            got = self.out_b.cpu().numpy()
            assert np.array_equal(got[told], b[told])
            assert np.array_equal(got[~told], self.born[~told] if self.in_place else b[~told])
        assert bool((self.workspace[self.args.workspace_bytes:] == 255).all())

    def check(self, ctx):
        self.upload()
        ctx.kv_evict_device(self.cache, self.args, sync=True)
        self.compare()
        return self


LENGTHS = [1, 2, 5, 63, 64, 65, 100, 128, 200, 257, 300, 7]


@pytest.mark.parametrize("born", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("part", [0.0, 0.1, 0.5, 0.9, 1.0])
def test_parts_of_sequences_stay(mit2, ctx, born, in_place, part):
    Cut(mit2, LENGTHS, [int(n * part) for n in LENGTHS], born=born, in_place=in_place, seed=int(part * 10)).check(ctx)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,page", [(32, 1, 1), (64, 5, 16), (96, 2, 8), (128, 3, 64), (192, 2, 4), (256, 1, 32)])
def test_types_heads_and_pages(mit2, ctx, dtype, dim, heads, page):
    Cut(mit2, [90, 40, 3], [50, 39, 3], heads=heads, dim=dim, page=page, dtype=dtype, born=True, seed=dim).check(ctx)


@pytest.mark.parametrize("length,keep", [(700, 699), (700, 636), (2100, 700), (3000, 2999), (5000, 1250), (8192, 4000), (8193, 8000), (20000, 9999)])
def test_long_sequences(mit2, ctx, length, keep):
    Cut(mit2, [length, length // 3], [keep, length // 4], layers=1, heads=2, page=64, first=4, last=100, born=length % 1000 == 700, seed=length).check(ctx)


@pytest.mark.parametrize("first,last", [(0, 0), (0, 50), (50, 0), (20, 30), (40, 60), (0, 1000), (1000, 0), (2 ** 32 - 1, 2 ** 32 - 1)])
@pytest.mark.parametrize("born", [False, True])
def test_protected_rows(mit2, ctx, first, last, born):
    """Also more of them than may stay: then the lowest places of those."""
    Cut(mit2, [120, 30], [50, 20], first=first, last=last, born=born, seed=first % 97 + last % 89).check(ctx)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "wild"])
@pytest.mark.parametrize("length", [150, 3000])
def test_equal_and_wild_weights(mit2, ctx, kind, length):
    rng = np.random.default_rng(4)
    shape = (1, 2, 2, length + 8)
    w = {"equal": np.full(shape, 0.25), "few": rng.integers(0, 3, shape) * 0.5, "zeros": np.where(rng.random(shape) < 0.5, -0.0, 0.0),
         "wild": rng.choice([np.nan, -np.nan, np.inf, -np.inf, 1e-45, -1e-45, 0.0, -0.0, 3e38, -3e38, 1.0, -1.0], shape)}[kind].astype(np.float32)
    Cut(mit2, [length, length - 20], [length // 2, 10], layers=1, weights=w, seed=1).check(ctx)


@pytest.mark.parametrize("in_place", [False, True])
def test_places_without_a_page(mit2, ctx, in_place):
    c = Cut(mit2, [100, 90, 60], [50, 80, 20], first=3, last=4, in_place=in_place, seed=5)
    c.table[0, 1], c.table[0, 9], c.table[1, 0], c.table[2, :] = -1, c.k.shape[1], 2 ** 31 - 1, -2 ** 31
    c.check(ctx)


def test_odd_lengths_and_budgets(mit2, ctx):
    """Past the table, past the weights, negative, none; budgets past the length, zero, negative."""
    c = Cut(mit2, [50, 50, 50, 50, 50, 50, 50], [20, 20, 20, 20, 60, 0, -4], seed=6)
    c.length = [100000, 2 ** 31 - 1, -3, 0, 50, 50, 50]
    c.check(ctx)
    for stride in (1, 33, 57):
        Cut(mit2, [50, 20], [20, 19], stride=stride, seed=7, born=True).check(ctx)


def test_births_at_the_ends_of_their_range(mit2, ctx):
    c = Cut(mit2, [40, 40], [12, 30], last=5, born=True, seed=8)
    rng = np.random.default_rng(1)
    c.born = rng.choice(np.array([-2 ** 31, -1, 0, 2 ** 31 - 1], np.int32), c.born.shape)
    c.now = np.array([-2 ** 31, 2 ** 31 - 1], np.int32)
    c.check(ctx)
    c.last = 2 ** 32 - 1
    c.check(ctx)


@pytest.mark.parametrize("hint", [0, 1, 100, 5000, 2 ** 32 - 1])
def test_any_length_hint(mit2, ctx, hint):
    Cut(mit2, [700, 30], [300, 29], hint=hint, seed=9).check(ctx)


@pytest.mark.parametrize("kind", ["any", "equal", "few", "wild"])
@pytest.mark.parametrize("length", [2, 64, 700, 1024, 1025, 4096, 8190, 16384, 17000])
def test_one_row_leaves(mit2, ctx, length, kind):
    """The last of the least, which may be the row behind the budget; of a hint of one wave's length too."""
    rng = np.random.default_rng(length)
    shape = (2, 3, 2, length)
    w = {"any": rng.exponential(1.0, shape), "equal": np.full(shape, 0.25), "few": rng.integers(0, 3, shape) * 0.5,
         "wild": rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0], shape)}[kind].astype(np.float32)
    w[0, 0, 0, length - 1] = -3e38
    lengths = [length, max(2, length // 2), max(2, length - 3)]
    for first, last, hint in ((0, 0, None), (1, 5, None), (2 ** 32 - 1, 0, None), (4, 0, 0)):
        Cut(mit2, lengths, [n - 1 for n in lengths], heads=2, page=64, weights=w, stride=length, first=first, last=last, hint=hint, seed=length).check(ctx)


@pytest.mark.parametrize("kind", ["any", "equal", "few", "wild"])
@pytest.mark.parametrize("length", [40, 64, 129, 700, 1024])
def test_few_rows_leave(mit2, ctx, length, kind):
    """2 to 33 of a line, those behind the budget among them; all protected, and some places without a page."""
    rng = np.random.default_rng(length)
    leave = [2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 32, 33]
    shape = (1, len(leave), 2, length)
    w = {"any": rng.exponential(1.0, shape), "equal": np.full(shape, 0.25), "few": rng.integers(0, 3, shape) * 0.5,
         "wild": rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0], shape)}[kind].astype(np.float32)
    w[:, :, 0, length - 6:] = -1.0  # (those behind the budget leave, with others or alone)
    for first, last, born in ((0, 0, False), (3, 4, False), (2 ** 32 - 1, 0, False), (1, 20, True)):
        c = Cut(mit2, [length] * len(leave), [length - r for r in leave], layers=1, heads=2, page=8, weights=w, stride=length, first=first, last=last, born=born,
                seed=length)
        if kind == "few":
            c.table[:, 2] = -1
        c.check(ctx)


def test_many_sequences_and_layers(mit2, ctx):
    length = [(7 * s) % 40 for s in range(150)]
    Cut(mit2, length, [n // 2 for n in length], layers=5, heads=3, seed=10).check(ctx)


def test_pages_below_the_first_rows_are_not_touched(mit2, ctx):
    """Sequences that share a prefix's pages: those stay as they are, and each sequence's rows are its own."""
    c = Cut(mit2, [80, 80, 80], [40, 33, 64], first=32, last=4, page=16, seed=11, in_place=True)
    c.table[1:, :2] = c.table[0, :2]
    c.check(ctx)
    for s in range(3):
        for p in c.table[s, :2]:
            assert torch.equal(c.dk[:, p].cpu(), c.k[:, p])


def test_cut_again_and_again(mit2, ctx):
    """Steps of a full cache: one row in, one row out, births kept in step; in place, as a decoder does it."""
    c = Cut(mit2, [60, 60], [59, 59], first=2, last=8, born=True, in_place=True, seed=12)
    c.now[:] = 200
    rng = np.random.default_rng(2)
    c.upload()
    for step in range(6):
        expect = context_ref.evict(c.dk.double().cpu().numpy(), c.dv.double().cpu().numpy(), c.table, c.page, [60, 60], c.keep, c.dw.cpu().numpy(), c.first,
                                   c.last, c.db.cpu().numpy(), c.now)
        ctx.kv_evict_device(c.cache, c.args, sync=True)
        assert np.array_equal(c.dk.double().cpu().numpy(), expect[0]) and np.array_equal(c.dv.double().cpu().numpy(), expect[1])
        assert np.array_equal(c.dw.cpu().numpy()[..., :59], expect[2][..., :59]) and np.array_equal(c.db.cpu().numpy()[..., :59], expect[3][..., :59])
        assert c.dl.cpu().tolist() == [59, 59]
        # the next step's row
        c.dl += 1
        c.now += 1
        c.dn += 1
        c.db[..., 59] = int(c.now[0]) - 1
        c.dw[..., 59] = torch.from_numpy(rng.random(c.weights.shape[:3]).astype(np.float32))
        torch.cuda.synchronize()


def test_nothing_to_do(mit2, ctx):
    c = Cut(mit2, [20], [5], seed=13)
    c.upload()
    c.args.seqs = 0
    ctx.kv_evict_device(c.cache, c.args, sync=True)
    assert torch.equal(c.dk.cpu(), c.k) and c.out_l.cpu().tolist() == [-9]


def test_the_lower_layers_of_a_larger_stride(mit2, ctx):
    """Layers with room between them, which is left alone."""
    c = Cut(mit2, [50, 30], [20, 10], layers=3, dtype="f16", seed=14)
    c.upload()
    size, gap = c.k[0].numel(), 64
    wide = [torch.full((3 * (size + gap),), 7.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    for flat, small in zip(wide, (c.k, c.v)):
        flat.view(3, -1)[:, :size] = small.reshape(3, -1).to(DEV)
    c.cache.k, c.cache.v = (x.data_ptr() for x in wide)
    c.args.layer_stride = size + gap
    torch.cuda.synchronize()
    ctx.kv_evict_device(c.cache, c.args, sync=True)
    k, v = c.expect()[:2]
    for flat, want in zip(wide, (k, v)):
        assert np.array_equal(flat.view(3, -1)[:, :size].double().cpu().numpy(), want.reshape(3, -1))
        assert bool((flat.view(3, -1)[:, size:] == 7.0).all())


def test_offsets_past_32_bits(mit2, ctx):
    """Rows move between pages over 2^32 elements in; weights of a layer over 2^31 elements in."""
    c = Cut(mit2, [100], [40], layers=1, heads=8, dim=128, page=64, dtype="bf16", seed=15)
    c.upload()
    pages, shift = 70000, 70000 - c.k.shape[1]
    big = [torch.empty(pages * 8 * 64 * 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    stride = 1 << 28
    far = torch.empty(8 * stride, device=DEV)
    try:
        for flat, small in zip(big, (c.k, c.v)):
            flat.view(pages, 8, 64, 128)[shift:] = small[0].to(DEV)
        for h in range(8):
            far[h * stride: h * stride + 100] = c.dw[0, 0, h, :100]
        c.dt += shift
        c.cache.k, c.cache.v, c.cache.pages = big[0].data_ptr(), big[1].data_ptr(), pages
        c.args.weights = c.args.weights_out = far.data_ptr()
        c.args.weight_stride = stride
        n = mit2.kv_evict_workspace(c.cache, c.args)
        room = torch.empty(n, dtype=torch.uint8, device=DEV)
        c.args.workspace, c.args.workspace_bytes = room.data_ptr(), n
        torch.cuda.synchronize()
        ctx.kv_evict_device(c.cache, c.args, sync=True)
        k, v, w, _, _ = c.expect()
        for flat, want in zip(big, (k, v)):
            assert np.array_equal(flat.view(pages, 8, 64, 128)[shift:].double().cpu().numpy(), want[0])
        for h in range(8):
            assert np.array_equal(far[h * stride: h * stride + 40].cpu().numpy(), w[0, 0, h, :40])
    finally:
        del big, far
        torch.cuda.empty_cache()


@pytest.mark.parametrize("length,hint", [(16500, 16500), (40000, 40000), (20000, 100000), (3000, 100000), (100, 1 << 30), (20000, 500), (20000, 3000)])
@pytest.mark.parametrize("born", [False, True])
def test_lines_in_segments_and_hints_that_are_off(mit2, ctx, length, hint, born):
    """Lines longer than a block holds, in segments; and shorter and longer ones than their launch was laid out for."""
    Cut(mit2, [length, length - 77, 5], [length // 2 + 3, length - 78, 2], layers=1, heads=1, page=128, first=5, last=60, born=born, hint=hint, seed=length,
        capacity=[max(length, hint) if hint < 1 << 20 else length]).check(ctx)


@pytest.mark.parametrize("kind", ["equal", "few", "wild"])
@pytest.mark.parametrize("part", [0.001, 0.5, 0.999])
def test_equal_and_wild_weights_in_segments(mit2, ctx, kind, part):
    rng = np.random.default_rng(5)
    shape = (1, 1, 2, 33000)
    w = {"equal": np.full(shape, 0.25), "few": rng.integers(0, 3, shape) * 0.5,
         "wild": rng.choice([np.nan, np.inf, -np.inf, 1e-45, -1e-45, 0.0, -0.0, 3e38, 1.0, 1.0000001, -1.0], shape)}[kind].astype(np.float32)
    Cut(mit2, [32900], [int(32900 * part)], layers=1, page=128, weights=w, seed=1).check(ctx)
