"""16-bit shared-prefix attention (mit2cfm_kv_prefix_attention_device) keeps its weights to twice the type's bits, however many query rows a group
or a sequence has: against 64 bits it is off by the result's rounding and by what fp32 leaves."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
import ops_ref  # noqa: E402
from context_ref import check, mine  # noqa: E402
from ops_ref import HALF_STEP, Batch  # noqa: E402
from test_gpu_kv_prefix import Shared, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# dim, heads, new rows, own rows, shared rows, page: one query tile a wave, two (heads of other sizes, groups of up to 32 query rows), the block form
# by its groups (tokens) and by its sequences, and sequences outside all groups
CASES = [(64, (4, 4), [1] * 9, [5, 40, 3], 300, 16), (64, (4, 2), [1] * 12, [50, 7, 129], 250, 64), (96, (6, 2), [1] * 20, [31, 2, 70], 200, 16),
         (256, (4, 1), [1] * 9, [9, 33, 60], 140, 32), (192, (4, 2), [12, 9, 17], [20, 77, 30], 130, 16), (32, (7, 1), [3, 8, 1], [90, 30, 2], 700, 8),
         (64, (20, 20), [1] * 40, [60, 3, 31], 260, 64), (128, (32, 8), [1] * 10, [100, 40, 7], 900, 16), (128, (8, 2), [9, 12, 7, 10], [40, 130, 1, 77], 320, 32),
         (64, (4, 2), [70, 1, 40], [7, 90, 200], 190, 16), (128, (4, 4), [90, 33, 64], [5, 260, 64], 400, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,new,own,shared,page", CASES)
@pytest.mark.parametrize("grouped", [True, False])
def test_weights_are_not_rounded_to_the_type(mit2, ctx, dtype, dim, heads, new, own, shared, page, grouped):  # noqa: F811
    length = [shared + n + own[s % len(own)] for s, n in enumerate(new)]
    b = Batch(new, length, page=page, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim + len(new))
    bounds, said = ([0, len(new)], [shared]) if grouped else ([len(new) - 1, len(new)], [shared])  # (most of them in no group)
    context_ref.share(b, bounds, said, True)
    mask = ops_ref.trees(b, 3)[0] if max(new) > 1 else None
    got = Shared(mit2, b, bounds, said, mask=mask).run(ctx)
    b.dtype = "f32"  # (the reference's tolerance as if nothing but fp32 were at work)
    ref, tol = ops_ref.attention64(b, dim ** -0.5, mask)
    value = b.v
    b.v = value.abs()
    spread = ops_ref.attention64(b, dim ** -0.5, mask)[0]  # sum of weight x |value|
    b.v = value
    # a weight's two parts: off by a half step of a half step of it; in f16 also by 2^-25, half its smallest number, where the largest weight is
    # at least 2^7.  Then the result's rounding.
    e = tol + HALF_STEP[dtype] ** 2 * spread + (max(length) * 2.0 ** -32 * float(value.abs().max()) if dtype == "f16" else 0.0)
    m = mine(b)
    check(got[m], ref[m], (e + HALF_STEP[dtype] * (ref.abs() + e))[m], f"weights {dtype} {dim}")
