"""The normed append (mit2cfm_kv_norm_append_device) on the GPU against a plain 64-bit restatement (context_ref.py)."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
from context_ref import DEV, On, check, mine  # noqa: E402
from ops_ref import TORCH, Batch  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(mit2):
    c = mit2.Context(synthetic_seed=3, device=0)
    yield c
    c.close()


def _weights(b, heads, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return [(1.0 + 0.3 * torch.randn(n, b.dim, generator=g)).to(TORCH[dtype]) for n in heads]


def _run(mit2, ctx, b, *, per_head=False, weights=True, weight_dtype=None, eps=1e-6, centered=False, position=None, rot=0, interleaved=False,
         theta=10000.0, what=""):
    on = On(mit2, b)
    a = on.append_args(position=position, rot=rot, interleaved=interleaved, theta=theta)
    wt = weight_dtype or b.dtype
    qw, kw = _weights(b, (b.q_heads, b.kv_heads) if per_head else (1, 1), 5, wt) if weights else (None, None)
    n = mit2.KvNorm(weight_dtype=mit2.DTYPES[wt], centered=int(centered), eps=eps)
    if weights:
        on.weights = qw.to(DEV), kw.to(DEV)
        n.q_weight, n.k_weight = (x.data_ptr() for x in on.weights)
        n.q_weight_head = n.k_weight_head = b.dim if per_head else 0
    torch.cuda.synchronize()
    ctx.kv_norm_append_device(on.cache, on.rows, a, n, sync=True)
    q, qt, k, kt, v = context_ref.norm_append64(b, qw, kw, n.eps, centered, position, rot, interleaved, theta)
    got = on.out.double().cpu()
    assert bool(torch.isnan(got[~mine(b)]).all()), "rows of no sequence were written"
    what = what or f"{b.dtype} {b.dim}/{rot}"
    check(got, q, qt, "q " + what)
    check(on.k.double().cpu(), k, kt, "k " + what)
    assert torch.equal(on.v.double().cpu(), v)
    return on, a, n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 0, False), (64, 64, True), (64, 64, False), (128, 96, False), (96, 32, True), (96, 96, False), (32, 10, False),
                                                 (32, 6, True), (32, 32, False), (256, 256, False), (192, 48, False), (192, 192, True)])
@pytest.mark.parametrize("centered", [False, True])
def test_heads_are_normed_and_rotated(mit2, ctx, dtype, dim, rot, interleaved, centered):
    b = Batch([1, 0, 5, 17, 2], [1, 0, 5, 40, 130], page=16, kv_heads=2, q_heads=6, dim=dim, dtype=dtype, seed=dim + rot, tail_rows=3, lead_rows=2)
    _run(mit2, ctx, b, rot=rot, interleaved=interleaved, centered=centered)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("weight_dtype", ["f32", None])
def test_weights(mit2, ctx, dtype, per_head, weight_dtype):
    b = Batch([3, 1], [3, 50], page=8, kv_heads=3, q_heads=9, dim=96, dtype=dtype, seed=2)
    _run(mit2, ctx, b, per_head=per_head, weight_dtype=weight_dtype, rot=64)
    _run(mit2, ctx, b, weights=False, rot=64)


@pytest.mark.parametrize("heads", [(20, 20), (1, 1), (7, 1), (70, 2)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_head_counts(mit2, ctx, heads, dtype):
    _run(mit2, ctx, Batch([2, 1], [9, 70], page=64, kv_heads=heads[1], q_heads=heads[0], dim=64, dtype=dtype, seed=7), rot=64)


def test_many_rows_and_sequences(mit2, ctx):
    """Rows enough that blocks take several passes, sequences more than a wave's lanes, some without rows."""
    new = [(7 * s) % 31 for s in range(150)]
    _run(mit2, ctx, Batch(new, [n + (11 * s) % 50 for s, n in enumerate(new)], page=8, kv_heads=1, q_heads=40, dim=64, dtype="bf16", seed=9, tail_rows=5),
         rot=64, interleaved=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("centered", [False, True])
def test_small_large_and_equal_elements(mit2, ctx, dtype, centered):
    """Heads of zeros, of one value, of elements whose squares leave fp32's range either way."""
    b = Batch([6], [9], dim=64, dtype=dtype, seed=3)
    top = {"f32": 2.0 ** 110, "f16": 2.0 ** 14, "bf16": 2.0 ** 110}[dtype]
    low = {"f32": 2.0 ** -100, "f16": 2.0 ** -20, "bf16": 2.0 ** -100}[dtype]
    for x in (b.q, b.new_k):
        x[0] = 0.0
        x[1] = 0.5
        x[2] *= top
        x[3] *= low
        x[4, :, ::2] *= top
    _run(mit2, ctx, b, rot=64, centered=centered)
    _run(mit2, ctx, b, rot=32, centered=centered, eps=1e-20, weights=False)


def test_elements_that_are_not_finite_stay_in_their_heads(mit2, ctx):
    b = Batch([4], [9], page=16, kv_heads=2, q_heads=4, dim=64, dtype="f32", seed=4)
    clean, _, _ = _run(mit2, ctx, b, rot=64)
    b.q[1, 2, 5], b.new_k[2, 1, 60] = math.nan, math.inf
    on = On(mit2, b)
    qw, kw = (x.to(DEV) for x in _weights(b, (1, 1), 5, "f32"))
    n = mit2.KvNorm(weight_dtype=mit2.DTYPES["f32"], eps=1e-6, q_weight=qw.data_ptr(), k_weight=kw.data_ptr())
    torch.cuda.synchronize()
    ctx.kv_norm_append_device(on.cache, on.rows, on.append_args(rot=64), n, sync=True)
    assert bool(torch.isnan(on.out[1, 2]).all())
    on.out[1, 2] = clean.out[1, 2]
    assert torch.equal(on.out, clean.out)
    page, at = b.page_of(0, 7), 7 % 16
    assert not bool(torch.isfinite(on.k[page, 1, at, 60]))
    on.k[page, 1, at] = clean.k[page, 1, at]
    assert torch.equal(on.k, clean.k)


def test_far_and_negative_positions(mit2, ctx):
    b = Batch([7], [9], dim=64, dtype="f32", seed=2)
    for theta in (10000.0, 500000.0):
        _run(mit2, ctx, b, rot=64, position=np.array([0, -3, 131071, 1000003, 16777217, 2147483647, -2147483648], np.int32), theta=theta)


def test_rows_without_a_page_are_dropped(mit2, ctx):
    b = Batch([4, 4, 3], [20, 36, 3], page=16, dim=64, dtype="f32", seed=4)
    b.table[0, 1], b.table[1, 2], b.table[2, 0] = -1, b.pages, 2 ** 31 - 1
    _run(mit2, ctx, b)
    b = Batch([2, 3], [2, 3], page=16, dim=64, dtype="f32", seed=5)
    b.length = [1, 100]  # before the sequence's begin; past its table
    _run(mit2, ctx, b, rot=64)


@pytest.mark.parametrize("pad", [8, 3])
def test_strides_in_place_and_without_queries(mit2, ctx, pad):
    """q, k and v as slices of one projection's rows (an odd row stride: element-wise), q in place; weights at an odd address; then no q."""
    b = Batch([3, 6], [3, 30], page=8, kv_heads=2, q_heads=4, dim=64, dtype="f16", seed=6)
    plain, a, n = _run(mit2, ctx, b, rot=64, interleaved=True)
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
    odd = torch.zeros(b.dim + 1, dtype=TORCH[b.dtype], device=DEV)
    odd[1:] = plain.weights[0][0]
    if pad == 3:
        n.q_weight = odd.data_ptr() + 2
    torch.cuda.synchronize()
    ctx.kv_norm_append_device(on.cache, on.rows, a, n, sync=True)
    # (the sums' order is the form's: a last bit of the type apart)
    step = torch.finfo(TORCH[b.dtype]).eps
    got = packed[:, : b.q_heads * b.dim].reshape(plain.out.shape).float()
    assert bool(((got - plain.out.float()).abs() <= step * plain.out.float().abs() + 1e-6).all())
    assert bool(((on.k.float() - plain.k.float()).abs() <= step * plain.k.float().abs() + 1e-6).all()) and torch.equal(on.v, plain.v)
    k = on.k.clone()
    a.q, a.q_out, a.q_heads = None, None, 0
    on.k.copy_(b.k)
    torch.cuda.synchronize()
    ctx.kv_norm_append_device(on.cache, on.rows, a, n, sync=True)
    assert torch.equal(on.k, k)


def test_norm_and_append_agree_with_the_plain_append(mit2, ctx):
    """Heads that are normalised already (weights 1, a mean square of 1): the plain append's rotation, to rounding."""
    b = Batch([5, 2], [40, 9], dim=128, dtype="f32", seed=8)
    for x in (b.q, b.new_k):
        x /= (x.double() ** 2).mean(-1, keepdim=True).sqrt().float()
    on, _, _ = _run(mit2, ctx, b, rot=128, weights=False, eps=1e-20)
    plain = On(mit2, b)
    ctx.kv_append_device(plain.cache, plain.rows, plain.append_args(rot=128), sync=True)
    assert float((on.out - plain.out).abs().max()) < 1e-5 and float((on.k - plain.k).abs().max()) < 1e-5


@pytest.mark.parametrize("seqs", [0, 2])
def test_nothing_to_do(mit2, ctx, seqs):
    b = Batch([1, 1], [4, 4], dim=64, dtype="f32", seed=15)
    on = On(mit2, b)
    on.rows.seqs, on.rows.rows = seqs, 0 if seqs else 2
    ctx.kv_norm_append_device(on.cache, on.rows, on.append_args(), mit2.KvNorm(eps=1e-6), sync=True)
    assert torch.equal(on.k.cpu(), b.k) and bool(torch.isnan(on.out).all())
