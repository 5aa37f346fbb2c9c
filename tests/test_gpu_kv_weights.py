"""16-bit attention of few query rows (mit2cfm_kv_attention_device: up to 16 rows x query heads of a key head, a sequence on average) keeps its
weights to twice the type's bits: against 64 bits it is off by the result's rounding and by what fp32 leaves."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import ops_ref  # noqa: E402
from ops_ref import HALF_STEP, Batch  # noqa: E402
from test_gpu_kv_ops import On, _check, _mine, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new,length,page", [(64, (20, 20), [1, 1, 1], [1, 33, 703], 64), (128, (32, 8), [1, 3], [900, 40], 16), (128, (8, 1), [1], [5000], 32),
                                                       (32, (7, 1), [2, 1], [90, 17], 8), (96, (24, 4), [2, 3], [300, 64], 32),
                                                       (64, (4, 4), [14, 12], [400, 55], 16), (256, (2, 1), [8], [130], 16), (192, (4, 2), [1, 7], [70, 600], 128)])
def test_weights_are_not_rounded_to_the_type(mit2, ctx, dtype, dim, heads, new, length, page):  # noqa: F811
    b = Batch(new, length, page=page, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim + len(new))
    mask = ops_ref.trees(b, 3)[0] if max(new) > 1 else None
    got = On(mit2, b).attend(ctx, mask=mask)
    b.dtype = "f32"  # (the reference's tolerance as if nothing but fp32 were at work)
    ref, tol = ops_ref.attention64(b, dim ** -0.5, mask)
    value = b.v
    b.v = value.abs()
    spread = ops_ref.attention64(b, dim ** -0.5, mask)[0]  # sum of weight x |value|
    b.v = value
    # a weight's two parts: off by a half step of a half step of it; in f16 also by 2^-25, half its smallest number, where the largest weight is
    # at least 2^7.  Then the result's rounding.
    e = tol + HALF_STEP[dtype] ** 2 * spread + (max(length) * 2.0 ** -32 * float(value.abs().max()) if dtype == "f16" else 0.0)
    mine = _mine(b)
    _check(got[mine], ref[mine], (e + HALF_STEP[dtype] * (ref.abs() + e))[mine], f"weights {dtype} {dim}")
