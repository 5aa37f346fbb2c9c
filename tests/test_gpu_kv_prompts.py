"""Paged attention over whole prompts and long chains (mit2cfm_kv_attention_device): many tiles of query rows, each seeing the rows before it."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ops_ref  # noqa: E402
from ops_ref import Batch  # noqa: E402
from test_gpu_kv_ops import On, _check, _check_attention, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,page", [(64, (2, 2), 64), (128, (4, 1), 16), (96, (2, 1), 32)])
@pytest.mark.parametrize("new,old", [([2047], [0]), ([600, 1, 1030], [0, 44, 333]), ([257, 256, 255, 1], [1000, 0, 17, 900])])
def test_prompts(mit2, ctx, dtype, dim, heads, page, new, old):  # noqa: F811
    b = Batch(new, [n + o for n, o in zip(new, old)], page=page, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=dim + len(new), tail_rows=2)
    _check_attention(ctx, mit2, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_prompt_in_pieces_is_the_prompt(mit2, ctx, dtype):  # noqa: F811
    """A prompt taken whole, and in pieces of 700 rows each over those before: the same within the tolerance of each."""
    whole = Batch([1900], [1900], page=64, q_heads=4, kv_heads=2, dim=128, dtype=dtype, seed=5)
    ref, tol = ops_ref.attention64(whole, 128 ** -0.5)
    _check(On(mit2, whole).attend(ctx), ref, tol, f"whole {dtype}")
    for first in range(0, 1900, 700):
        n = min(700, 1900 - first)
        piece = Batch([n], [first + n], page=64, q_heads=4, kv_heads=2, dim=128, dtype=dtype, seed=5)
        piece.k, piece.v, piece.pages, piece.table = whole.k, whole.v, whole.pages, whole.table.copy()
        piece.q = whole.q[first: first + n].clone()
        _check(On(mit2, piece).attend(ctx), ref[first: first + n], tol[first: first + n], f"piece at {first} {dtype}")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_a_large_tree(mit2, ctx, dtype):  # noqa: F811
    """More new rows than a mask's words hold in one tile, over a cache, with rows that see nothing of the tree."""
    b = Batch([700, 33], [1000, 40], page=32, q_heads=4, kv_heads=2, dim=64, dtype=dtype, seed=6)
    mask = ops_ref.trees(b, 8)[0]
    mask[[0, 31, 640, 699]] = 0
    _check_attention(ctx, mit2, b, mask=np.ascontiguousarray(mask))
