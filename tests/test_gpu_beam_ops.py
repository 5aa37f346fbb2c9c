"""The beam operators (mit2cfm_beam_select_device, mit2cfm_beam_reorder_device) on the GPU against plain restatements
(ops_ref.py): ties, beams that do not exist yet or are finished, rows without a finite logit, bad parents and pages,
part pages, and a small search run with all four operators."""
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
