"""Scores of the beam selection (mit2cfm_beam_select_device) where logits are so large that 64 bits hold little beside them."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import ops_ref  # noqa: E402
from ops_ref import TORCH  # noqa: E402
from test_gpu_beam_ops import _check_select, _select, ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 700, 9001])
def test_a_beam_s_score_survives_infinite_and_huge_logits(mit2, ctx, dtype, vocab):  # noqa: F811
    """One logit at +inf (which counts as fp32's largest), or far above the others: the beam goes on at its own score, not at 0."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(2, 4, vocab, generator=g) * 2.5
    top = float(torch.finfo(TORCH[dtype]).max)
    x[0, 1, 17] = math.inf
    x[0, 2, 7] = min(1e30, top)
    x[0, 3, vocab - 1] = min(1e25, top / 2)
    x[1, 0, 3], x[1, 0, 4] = math.inf, 1.0
    x[1, 3, 0] = top
    scores = np.array([[-5.0, -1.25, -0.5, -9.75], [-0.125, -3.5, -40.0, -2.0]], np.float32)
    for count in (1, 2, 3, 8, 20):
        _check_select(mit2, ctx, x, scores, count, dtype=dtype)
    got = _select(mit2, ctx, x.to(TORCH[dtype]), scores, 2, dtype=dtype)
    assert got[0][0].tolist() == [-0.5, -1.25] and got[1][0].tolist() == [2, 1] and got[2][0].tolist() == [7, 17]
    assert got[0][1].tolist() == [-0.125, -2.0] and got[1][1].tolist() == [0, 3] and got[2][1].tolist() == [3, 0]


def test_equal_scores_of_one_beam_go_by_their_logits(mit2, ctx):  # noqa: F811
    """Beside a logit of 1e30 all others of the beam score alike in 64 bits: the larger logits come first, of equal ones the lowest token, wherever
    they lie in the row; and a beam's come before the next beam's."""
    x = torch.zeros(1, 2, 12000)
    x[0, :, 11999], x[0, :, 5000], x[0, :, 8500], x[0, :, 100] = 1e30, 2.0, 2.0, 1.0
    for count in (2, 3, 4, 6, 9):
        got = _select(mit2, ctx, x, np.array([[-1.0, -2.0]], np.float32), count)
        assert got[2][0].tolist() == [11999, 11999, 5000, 8500, 100, 0, 1, 2, 3][:count], count
        assert got[1][0].tolist() == [0, 1, 0, 0, 0, 0, 0, 0, 0][:count]
        assert got[0][0].tolist() == [-1.0, -2.0] + [float(np.float32(-1e30))] * (count - 2)
