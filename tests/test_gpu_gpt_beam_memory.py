"""What GPU memory a beam search of mel codes (mit2cfm_gpt_kv_beam) takes: its own sizes' worth, whatever was searched before."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

W, LAYERS, PAGE = 1280, 2, 64


@pytest.fixture
def ctx2(mit2, tensors):
    c = mit2.Context({**tensors, **mit2.synthetic_gpt_tensors(layers=LAYERS)}, device=0)
    yield c
    c.close()


def _prefix(n):
    return (np.random.default_rng(n).standard_normal((n, W)) * 0.05).astype(np.float32)


def _pages(rows, beams=1):
    """Bytes of `beams` sequences' fp32 pages for that many rows."""
    return 2 * LAYERS * beams * -(-rows // PAGE) * PAGE * W * 4


def _taken(call):
    """How much less GPU memory is free after a call."""
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    call()
    torch.cuda.synchronize()
    return before - torch.cuda.mem_get_info()[0]


def test_a_long_prefix_after_many_beams_takes_what_one_beam_needs(ctx2):
    """Eight beams over a short prefix, then one over a long one: not eight times the long one's pages."""
    P, steps = 6000, 8
    alone = {b: ctx2.gpt_kv_beam(_prefix(20), 5, b) for b in (8, 1)}
    ctx2.gpt_kv_greedy(_prefix(P), 1)  # (the decoder's own buffers for that prefix)
    taken = _taken(lambda: ctx2.gpt_kv_beam(_prefix(P), steps, 1))
    print(f"one beam of {P} rows took {taken / 1e6:.0f} MB more; its pages {_pages(P + steps) / 1e6:.0f} MB", flush=True)
    assert taken <= 2 * _pages(P + steps)
    for b, first in alone.items():  # both sizes again, in what is held now
        again = ctx2.gpt_kv_beam(_prefix(20), 5, b)
        assert [h.tolist() for h in again["predicted"]] == [h.tolist() for h in first["predicted"]]
        assert again["scores"].tolist() == first["scores"].tolist()
