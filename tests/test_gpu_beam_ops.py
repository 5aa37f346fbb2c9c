"""The beam operators (mit2cfm_beam_select_device, mit2cfm_beam_reorder_device) on the GPU against plain restatements
(ops_ref.py): ties, beams that do not exist yet or are finished, rows without a finite logit, bad parents and pages,
part pages, and a small search run with all four operators, eager and as a graph."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ops_ref  # noqa: E402
from ops_ref import TORCH, U  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx(mit2):
    c = mit2.Context(synthetic_seed=3, device=0)
    yield c
    c.close()


def _select(mit2, ctx, logits, scores, count, finished=None, stop=-1, row=None, dtype="f32"):
    """beam_select of a CPU tensor's logits; the outputs as numpy arrays."""
    n, b, v = logits.shape
    row = v if row is None else row
    wide = torch.full((n * b, row), math.nan, dtype=TORCH[dtype])
    wide[:, :v] = logits.reshape(n * b, v)
    wide = wide.to(DEV)
    sc = torch.as_tensor(scores, dtype=torch.float32, device=DEV)
    fin = None if finished is None else torch.as_tensor(finished, dtype=torch.int32, device=DEV)
    out = [torch.full((n * count + 1,), -77, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32, torch.int32)]
    a = mit2.BeamSelect(logits=wide.data_ptr(), logits_row=row, dtype=mit2.DTYPES[dtype], groups=n, beams=b, vocab=v, count=count,
                        scores=sc.data_ptr(), finished=None if fin is None else fin.data_ptr(), stop_token=stop, scores_out=out[0].data_ptr(),
                        parent_out=out[1].data_ptr(), token_out=out[2].data_ptr(), finished_out=out[3].data_ptr())
    need = mit2.beam_select_workspace(a)
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    torch.cuda.synchronize()
    ctx.beam_select_device(a, sync=True)
    assert bool((ws[need:] == 255).all()) and all(float(o[-1]) == -77 for o in out)
    return [o[:-1].view(n, count).cpu().numpy() for o in out]


def _check_select(mit2, ctx, logits, scores, count, finished=None, stop=-1, dtype="f32", row=None):
    logits = logits.to(TORCH[dtype])
    got = _select(mit2, ctx, logits, scores, count, finished, stop, row, dtype)
    ref = ops_ref.select64(logits.double().numpy(), np.asarray(scores, np.float32).astype(np.float64), count, finished, stop)
    for name, x, y in zip(("parent", "token", "finished"), got[1:], ref[1:]):
        assert np.array_equal(x, y), (name, x, y)
    fin = np.isfinite(ref[0])
    assert np.array_equal(fin, np.isfinite(got[0])) and np.array_equal(got[0][~fin], ref[0][~fin])
    # the sum's terms are each off by a few fp32 ulp of themselves and by the argument's rounding: under the softmax a mean |x - max| of at most
    # ln(vocab) + 1; then one rounding of the score
    tol = (math.log(logits.shape[2]) + 8) * 2 * U + U * np.abs(ref[0][fin])
    assert (np.abs(got[0][fin] - ref[0][fin]) <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,count", [(1, 1, 1, 1), (1, 1, 7, 7), (1, 3, 8194, 6), (5, 2, 100, 3), (2, 8, 1025, 16), (3, 4, 64, 64),
                                                      (1, 64, 300, 64), (2, 1, 50001, 32), (40, 3, 255, 4), (1, 5, 20000, 1), (2, 2, 40, 64)])
def test_select(mit2, ctx, dtype, groups, beams, vocab, count):
    g = torch.Generator().manual_seed(vocab)
    scores = -4 * torch.rand(groups, beams, generator=g).numpy()
    _check_select(mit2, ctx, torch.randn(groups, beams, vocab, generator=g) * 2.5, scores, count, dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_select_ties_go_to_the_lowest(mit2, ctx, dtype):
    flat = torch.zeros(2, 3, 500)
    _check_select(mit2, ctx, flat, np.zeros((2, 3)), 9, dtype=dtype)
    flat[0, 1, 100:140] = 2.0
    flat[1, :, ::7] = 1.0
    flat[1, :, 3] = -0.0
    _check_select(mit2, ctx, flat, np.zeros((2, 3)), 12, dtype=dtype)
    _check_select(mit2, ctx, torch.zeros(1, 2, 30000), np.zeros((1, 2)), 64, dtype=dtype)
    steps = torch.arange(30000).float().div(1000).floor().view(1, 1, -1)
    _check_select(mit2, ctx, steps, np.zeros((1, 1)), 64, dtype=dtype)
    _check_select(mit2, ctx, -steps, np.zeros((1, 1)), 64, dtype=dtype)


def test_select_first_step_and_finished_beams(mit2, ctx):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 4, 900, generator=g)
    first = np.full((3, 4), -np.inf, np.float32)
    first[:, 0] = 0.0
    _check_select(mit2, ctx, x, first, 8, stop=899)
    done = np.array([[0, 1, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0]], np.int32)
    scores = np.array([[-1, -0.5, -2, -90], [-3, -1, -2, -1], [0, -1, -2, -np.inf]], np.float32)
    _check_select(mit2, ctx, x, scores, 8, finished=done, stop=5)
    _check_select(mit2, ctx, x, scores, 4, finished=done * 7, stop=0)
    _check_select(mit2, ctx, x, np.full((3, 4), -np.inf, np.float32), 6, finished=done, stop=899)
    x[2, 1, 5] = 20.0
    _check_select(mit2, ctx, x, scores, 5, finished=done, stop=5)


def test_select_of_masked_and_odd_logits(mit2, ctx):
    """Forbidden codes at -inf or the type's lowest value, rows without a finite logit, NaN, +inf."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 700, generator=g)
    x[0, 0, 3:] = -math.inf
    x[0, 1] = -math.inf
    x[0, 2, :600] = torch.finfo(torch.float32).min
    x[1, 0, 7], x[1, 0, 9] = math.nan, -math.inf
    x[1, 1] = math.nan
    x[1, 2, 4] = math.inf
    _check_select(mit2, ctx, x, np.zeros((2, 3)), 10, dtype="f32")
    x[1] = -math.inf
    _check_select(mit2, ctx, x, np.zeros((2, 3)), 10, dtype="f32")
    x = torch.randn(1, 2, 700, generator=g)
    x[0, 0, 5:] = torch.finfo(torch.float16).min
    x[0, 1, 650] = math.inf
    _check_select(mit2, ctx, x, np.zeros((1, 2)), 10, dtype="f16")


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_select_orders_infinities_before_the_largest_finite(mit2, ctx, dtype):
    """Many logits at the type's largest finite value, a few at +inf (which counts as fp32's largest): those come first."""
    x = torch.full((1, 2, 900), torch.finfo(TORCH[dtype]).max)
    x[0, 0, ::64] = math.inf
    x[0, 1, [3, 500, 777]] = math.inf
    x[0, 1, 100:400] = 0.0
    for count in (2, 5, 20, 64):
        _check_select(mit2, ctx, x, np.zeros((1, 2)), count, dtype=dtype)


def test_select_row_stride_and_large_values(mit2, ctx):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 3, 333, generator=g) * 1000 + 50000
    for row in (333, 334, 336, 401):
        _check_select(mit2, ctx, x, -1e4 * np.ones((2, 3)), 6, row=row)
        _check_select(mit2, ctx, x / 4, np.zeros((2, 3)), 6, row=row, dtype="bf16")


# ------------------------------------------------------------------ reorder
def _reorder(mit2, ctx, k, v, table, page, parent, length, state=None, token=None, place=None):
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    groups, beams, entries = table.shape
    # (the type does not matter to a copy: 16-bit patterns for 2-byte caches)
    dk, dv, dt, dp, dl = dev(k), dev(v), dev(table), dev(parent), dev(length)
    ds, dtok, dpl = dev(state), dev(token), dev(place)
    out, so = torch.full_like(dt, -9), None if state is None else torch.full_like(ds, -9)
    cache = mit2.KvCache(k=at(dk), v=at(dv), table=at(dt), pages=k.shape[1], page_rows=page, kv_heads=k.shape[2], head_dim=k.shape[4],
                         table_stride=entries, dtype=mit2.DTYPE_F32 if k.itemsize == 4 else mit2.DTYPE_F16)
    a = mit2.BeamReorder(groups=groups, beams=beams, layers=k.shape[0], layer_stride=k[0].size, parent=at(dp), parent_stride=parent.shape[1],
                         length=at(dl), table_out=at(out), state=at(ds), state_out=at(so), state_words=0 if state is None else state.shape[2],
                         token=at(dtok), place=at(dpl))
    torch.cuda.synchronize()
    ctx.beam_reorder_device(cache, a, sync=True)
    return out.cpu().numpy(), dk.cpu().numpy(), dv.cpu().numpy(), None if so is None else so.cpu().numpy()


def _case(rng, groups, beams, entries, page, heads=2, dim=32, layers=2, kind=np.float32, words=9):
    pages = groups * beams * entries + 2
    shape = (layers, pages, heads, page, dim)
    k, v = (rng.integers(0, 30000, shape).astype(kind) for _ in range(2))
    table = rng.permutation(pages)[: groups * beams * entries].reshape(groups, beams, entries).astype(np.int32)
    return dict(k=k, v=v, table=table, page=page, state=rng.integers(0, 9000, (groups, beams, words)).astype(np.int32),
                token=rng.integers(0, 9000, (groups, beams)).astype(np.int32), place=rng.integers(0, words, groups).astype(np.int32))


def _same(got, ref):
    for name, x, y in zip(("table", "k", "v", "state"), got, ref):
        assert (x is None) == (y is None) and (x is None or np.array_equal(x, y)), name


@pytest.mark.parametrize("kind", [np.float32, np.int16])
@pytest.mark.parametrize("groups,beams,page,entries", [(1, 1, 16, 3), (1, 3, 16, 4), (4, 8, 8, 5), (2, 64, 4, 3), (3, 33, 1, 6), (1, 2, 128, 1)])
def test_reorder(mit2, ctx, kind, groups, beams, page, entries):
    rng = np.random.default_rng(beams + page)
    for n in sorted({0, 1, page - 1, page, page + 1, 2 * page + page // 2, entries * page - 1, entries * page}):
        if not 0 <= n <= entries * page:
            continue
        c = _case(rng, groups, beams, entries, page, kind=kind)
        parent = rng.integers(0, beams, (groups, beams)).astype(np.int32)
        length = np.full(groups, n, np.int32)
        _same(_reorder(mit2, ctx, parent=parent, length=length, **c), ops_ref.reorder(parent=parent, length=length, **c))


def test_reorder_keeps_every_private_page(mit2, ctx):
    """Over many steps, the beams' private pages stay a permutation of what they were, and their rows those of their histories."""
    rng = np.random.default_rng(5)
    c = _case(rng, 2, 6, 4, 8)
    c["state"] = None
    c["token"] = c["place"] = None
    for n in range(1, 20):
        parent = rng.integers(0, 6, (2, 6)).astype(np.int32)
        length = np.full(2, n, np.int32)
        ref = ops_ref.reorder(parent=parent, length=length, **c)
        got = _reorder(mit2, ctx, parent=parent, length=length, **c)
        _same(got, ref)
        full = n // 8
        for g in range(2):
            assert sorted(got[0][g, :, full:].ravel()) == sorted(c["table"][g, :, full:].ravel())
        c["table"], c["k"], c["v"] = got[:3]


def test_reorder_of_bad_parents_lengths_pages_and_places(mit2, ctx):
    rng = np.random.default_rng(6)
    c = _case(rng, 4, 5, 3, 8)
    c["table"][0, :, 1] = -1
    c["table"][1, 2, 1], c["table"][1, 3, 1] = 2 ** 31 - 1, -2 ** 31
    c["place"] = np.array([-1, 9, 2 ** 31 - 1, 8], np.int32)
    parent = np.array([[0, 0, 0, 4, 4], [2, 2, 3, 3, 1], [-1, 5, 0, 2 ** 31 - 1, -2 ** 31], [4, 3, 2, 1, 0]], np.int32)
    for length in ([12, 12, 12, 12], [-1, 25, 2 ** 31 - 1, 24]):
        length = np.array(length, np.int32)
        _same(_reorder(mit2, ctx, parent=parent, length=length, **c), ops_ref.reorder(parent=parent, length=length, **c))


def test_reorder_takes_a_longer_selection(mit2, ctx):
    """Parents and tokens of a selection of 2 x beams: the first `beams` of each group."""
    rng = np.random.default_rng(7)
    c = _case(rng, 3, 4, 3, 8)
    parent = rng.integers(0, 4, (3, 8)).astype(np.int32)
    c["token"] = rng.integers(0, 9000, (3, 8)).astype(np.int32)
    length = np.array([3, 9, 20], np.int32)
    _same(_reorder(mit2, ctx, parent=parent, length=length, **c), ops_ref.reorder(parent=parent, length=length, **c))


# ------------------------------------------------------------------ together
class Search:
    """A search over a toy model: a token's query, keys and values are rows of tables, and the attention's output is its logits.  Layer 1 of the
    cache takes keys and values the other way round and is read at the end alone."""
    GROUPS, BEAMS, HEADS, DIM, VOCAB, PAGE, ENTRIES, STEPS, START, STOP = 2, 3, 2, 32, 60, 4, 6, 10, 7, 11
    PREFIX = (5, 8)

    def __init__(self, mit2, ctx):
        self.mit2, self.ctx = mit2, ctx
        g = torch.Generator().manual_seed(41)
        n, d = self.GROUPS * self.BEAMS, self.DIM
        self.emb = [torch.randn(self.VOCAB, h * d, generator=g) * f for h, f in ((self.HEADS, 2.0), (1, 1.0), (1, 3.0))]  # q, k, v
        self.prefix = [[torch.randn(p, d, generator=g) for _ in range(2)] for p in self.PREFIX]
        self.pages = n * self.ENTRIES
        z = dict(device=DEV)
        self.tables = [e.to(DEV) for e in self.emb]
        self.q, self.k, self.v = (torch.zeros(n, h * d, **z) for h in (self.HEADS, 1, 1))
        self.qr, self.logits = torch.zeros(n, self.HEADS * d, **z), torch.zeros(n, self.HEADS * d, **z)
        self.cache_k, self.cache_v = (torch.zeros(2, self.pages, 1, self.PAGE, d, **z) for _ in range(2))
        ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, **z)  # noqa: E731
        self.start = torch.arange(n + 1, dtype=torch.int32, **z)
        self.length, self.glength, self.place = ints(n), ints(self.GROUPS), ints(self.GROUPS)
        self.token, self.parent = ints(n), ints(n)
        self.score, self.done = [torch.zeros(n, **z) for _ in range(2)], [ints(n) for _ in range(2)]
        self.table, self.hist = [ints(n, self.ENTRIES) for _ in range(2)], [ints(n, self.STEPS) for _ in range(2)]
        self.ws = torch.zeros(1 << 20, dtype=torch.uint8, **z)
        self.stream = torch.cuda.ExternalStream(ctx.stream)

    def cache(self, layer, side):
        return self.mit2.KvCache(k=self.cache_k[layer].data_ptr(), v=self.cache_v[layer].data_ptr(), table=self.table[side].data_ptr(),
                                 pages=self.pages, page_rows=self.PAGE, kv_heads=1, head_dim=self.DIM, table_stride=self.ENTRIES,
                                 dtype=self.mit2.DTYPE_F32)

    def append(self, layer, side, rows, k, v, rot, **q):
        self.ctx.kv_append_device(self.cache(layer, side), rows, self.mit2.KvAppend(
            k=k.data_ptr(), v=v.data_ptr(), k_row=self.DIM, k_head=self.DIM, v_row=self.DIM, v_head=self.DIM, rotary_dim=rot, theta=10000.0, **q))

    def move(self, side, state=True):
        h = self.hist
        self.ctx.beam_reorder_device(self.cache(0, side), self.mit2.BeamReorder(
            groups=self.GROUPS, beams=self.BEAMS, layers=2, layer_stride=self.cache_k[0].numel(), parent=self.parent.data_ptr(),
            parent_stride=self.BEAMS, length=self.glength.data_ptr(), table_out=self.table[1 - side].data_ptr(),
            state=h[side].data_ptr() if state else None, state_out=h[1 - side].data_ptr() if state else None, state_words=self.STEPS,
            token=self.token.data_ptr() if state else None, place=self.place.data_ptr()))

    def begin(self):
        """Every group's prefix in its first beam's pages, the other beams its children."""
        with torch.cuda.stream(self.stream):
            for t in (self.cache_k, self.cache_v, *self.hist, *self.done, self.parent, self.place):
                t.zero_()
            self.table[1].copy_(torch.arange(self.pages, dtype=torch.int32).view(-1, self.ENTRIES))
            self.score[0].fill_(-math.inf)
            self.score[0][:: self.BEAMS] = 0.0
            self.token.fill_(self.START)
            self.glength.copy_(torch.tensor(self.PREFIX, dtype=torch.int32))
            self.length.copy_(torch.tensor(self.PREFIX, dtype=torch.int32).repeat_interleave(self.BEAMS))
            bounds = [torch.tensor([0, p], dtype=torch.int32, device=DEV) for p in self.PREFIX]
            kv = [[t.to(DEV) for t in pair] for pair in self.prefix]
            self.stream.synchronize()
            for grp, p in enumerate(self.PREFIX):
                rows = self.mit2.KvRows(start=bounds[grp].data_ptr(), length=self.glength[grp:].data_ptr(), seqs=1, rows=p, max_length=p)
                whole, self.table[1] = self.table[1], self.table[1][grp * self.BEAMS:]
                self.append(0, 1, rows, *kv[grp], self.DIM)
                self.append(1, 1, rows, *kv[grp][::-1], 0)
                self.table[1] = whole
            self.move(1, state=False)
            self.stream.synchronize()

    def step(self, side):
        m, n, d = self.mit2, self.GROUPS * self.BEAMS, self.DIM
        with torch.cuda.stream(self.stream):
            self.length.add_(1)
            self.glength.add_(1)
            for t, to in zip(self.tables, (self.q, self.k, self.v)):
                torch.index_select(t, 0, self.token, out=to)
            rows = m.KvRows(start=self.start.data_ptr(), length=self.length.data_ptr(), seqs=n, rows=n, max_length=self.PAGE * self.ENTRIES)
            wide = dict(q_row=self.HEADS * d, q_head=d, q_heads=self.HEADS)
            self.append(0, side, rows, self.k, self.v, d, q=self.q.data_ptr(), q_out=self.qr.data_ptr(), q_out_row=self.HEADS * d, q_out_head=d, **wide)
            self.append(1, side, rows, self.v, self.k, 0)
            self.ctx.kv_attention_device(self.cache(0, side), rows, m.KvAttention(
                q=self.qr.data_ptr(), out=self.logits.data_ptr(), out_row=self.HEADS * d, out_head=d, scale=d ** -0.5,
                workspace=self.ws.data_ptr(), workspace_bytes=self.ws.numel(), **wide))
            self.ctx.beam_select_device(m.BeamSelect(
                logits=self.logits.data_ptr(), logits_row=self.HEADS * d, dtype=m.DTYPE_F32, groups=self.GROUPS, beams=self.BEAMS, vocab=self.VOCAB,
                count=self.BEAMS, scores=self.score[side].data_ptr(), finished=self.done[side].data_ptr(), stop_token=self.STOP,
                scores_out=self.score[1 - side].data_ptr(), parent_out=self.parent.data_ptr(), token_out=self.token.data_ptr(),
                finished_out=self.done[1 - side].data_ptr(), workspace=self.ws.data_ptr(), workspace_bytes=self.ws.numel()))
            self.move(side)
            self.place.add_(1)

    def result(self):
        self.stream.synchronize()
        return self.hist[0].cpu().clone(), self.score[0].cpu().clone(), self.cache_k.cpu().clone(), self.cache_v.cpu().clone(), self.table[0].cpu().clone()


def test_a_search_of_all_four_operators(mit2, ctx):
    """Every hypothesis' score is that of its own history, recomputed in 64 bits from nothing but the history, and both layers' caches hold it;
    replays of the steps as a graph, with the search begun anew in between, give the same bits."""
    from test_gpu_kv_ops import Graph
    s = Search(mit2, ctx)
    s.begin()
    for i in range(s.STEPS):
        s.step(i & 1)
    first = s.result()
    hist, score, ck, cv, table = first
    q_emb, k_emb, v_emb = (e.double() for e in s.emb)
    for r in range(s.GROUPS * s.BEAMS):
        grp, told = r // s.BEAMS, hist[r].tolist()
        P, total = s.PREFIX[grp], 0.0
        inputs = [s.START] + told[:-1]
        keys = [ops_ref.rotate64(x.view(1, -1), i, s.DIM, False, 10000.0)[0] for i, x in enumerate(s.prefix[grp][0])]
        vals = list(s.prefix[grp][1].double())
        for i, (x, t) in enumerate(zip(inputs, told)):
            keys.append(ops_ref.rotate64(k_emb[x].view(1, -1), P + i, s.DIM, False, 10000.0)[0])
            vals.append(v_emb[x])
            if s.STOP in told[:i]:
                assert t == s.STOP
                continue
            q = ops_ref.rotate64(q_emb[x].view(s.HEADS, -1), P + i, s.DIM, False, 10000.0)
            out = torch.softmax(q @ torch.stack(keys).t() * s.DIM ** -0.5, -1) @ torch.stack(vals)
            total += float(torch.log_softmax(out.reshape(-1)[: s.VOCAB], -1)[t])
        # a score of the attention is off by 8 fp32 half steps of sum |q k| (the turns' and the sums'), at most about 2 * 32 * 2 * scale = 23 here; an
        # output by twice that of values up to 12; a log probability by twice that, a step
        assert abs(total - float(score[r])) <= s.STEPS * 2 * 12 * 2 * 8 * 23 * U, (r, total, float(score[r]))
        for j in range(P + s.STEPS):
            page, slot = int(table[r, j // s.PAGE]), j % s.PAGE
            x = s.prefix[grp] if j < P else None
            k1, v1 = (x[1][j], x[0][j]) if j < P else (s.emb[2][inputs[j - P]], s.emb[1][inputs[j - P]])
            assert torch.equal(ck[1, page, 0, slot], k1) and torch.equal(cv[1, page, 0, slot], v1), (r, j)
            assert (ck[0, page, 0, slot].double() - keys[j]).abs().max() <= 8 * U * 5 and torch.equal(cv[0, page, 0, slot].double(), vals[j])
    assert len({tuple(h) for h in hist[: s.BEAMS].tolist()}) == s.BEAMS

    def pair():
        s.step(0)
        s.step(1)

    torch.cuda.synchronize()
    g = Graph(ctx, pair)
    try:
        for _ in range(3):
            s.begin()
            for _ in range(s.STEPS // 2):
                g.replay()
            for a, b in zip(first, s.result()):
                assert torch.equal(a, b)
    finally:
        g.close()
