"""Beam search of mel codes (mit2cfm_gpt_kv_beam), which runs on the paged-cache and beam operators, against a plain search over the
CPU oracle's single-row decode; one beam against the greedy decode; and calls of other sizes, or too large, in between."""
from __future__ import annotations

import math

import numpy as np
import pytest

import ops_ref

pytestmark = pytest.mark.gpu

W = 1280
# A step's log probabilities: both sides sum in fp32, over at most 5120 products, through 2 layers and the head (8 products
# in a row).  Roundings of either sign add up as their square root: 8 * sqrt(5120) * 2^-24 of sums of the logits' size (about 1).
STEP_TOL = 8 * math.sqrt(5120) * 2.0 ** -24


@pytest.fixture(scope="module")
def gpt2_t(mit2):
    return mit2.synthetic_gpt_tensors(layers=2)


@pytest.fixture(scope="module")
def ctx2(mit2, tensors, gpt2_t):
    c = mit2.Context({**tensors, **gpt2_t}, device=0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def orc2(orc, gpt2_t):
    return orc.GPT(gpt2_t)


def _prefix(n, seed):
    return (np.random.default_rng(seed).standard_normal((n, W)) * 0.05).astype(np.float32)


def _oracle_beams(orc2, gpt2_t, prefix, steps, beams, hf, start=8192, stop=8193):
    """The same search with every hypothesis' logits from the oracle; the smallest gap between a kept and a dropped candidate."""
    emb, pos = (gpt2_t[k].astype(np.float32) for k in ("gpt.mel_embedding.weight", "gpt.mel_pos_embedding.emb.weight"))
    hyps, scores, done = [[start]] * beams, np.full(beams, -np.inf), np.zeros(beams, np.int32)
    scores[0] = 0.0
    gap = math.inf
    for step in range(steps):
        logits = np.full((1, beams, 8194), -np.inf)
        for b in range(beams):
            if scores[b] > -np.inf and not done[b]:
                rows = [emb[t] + pos[s + 1 if hf and s else s] for s, t in enumerate(hyps[b])]
                logits[0, b] = orc2.cached_decode(np.concatenate([prefix, np.stack(rows)]), prefix.shape[0] + step)[2]
        sc, parent, token, fin = ops_ref.select64(logits, scores[None], beams + 1, done[None], stop)
        gap = min(gap, float(sc[0, beams - 1] - sc[0, beams]))
        hyps = [hyps[p] + [int(t)] for p, t in zip(parent[0, :beams], token[0, :beams])]
        scores, done = sc[0, :beams], fin[0, :beams].astype(np.int32)
        if done.all():
            break
    cut = [h[1: h.index(stop) + 1] if stop in h else h[1:] for h in hyps]
    return cut, scores, gap


@pytest.mark.parametrize("P,steps,beams,hf", [(0, 3, 3, False), (5, 4, 3, True), (63, 3, 2, False), (64, 3, 4, True), (130, 9, 3, False),
                                              (20, 2, 8, False), (7, 5, 1, True)])
def test_beam_search_matches_the_oracle(ctx2, orc2, gpt2_t, P, steps, beams, hf):
    prefix = _prefix(P, P + 1)
    got = ctx2.gpt_kv_beam(prefix, steps, beams, hf)
    ref, scores, gap = _oracle_beams(orc2, gpt2_t, prefix, steps, beams, hf)
    print(f"beams {beams} P={P} steps={steps}: scores {got['scores']} / {scores}, smallest gap {gap:.2e}", flush=True)
    tol = STEP_TOL * steps + 2.0 ** -24 * np.abs(scores).max()  # (and the score's own rounding)
    assert np.abs(got["scores"] - scores).max() <= tol
    if gap > 2 * tol:
        assert [h.tolist() for h in got["predicted"]] == ref
    else:  # candidates too near each other to tell: the same number of tokens, scores as above
        assert [len(h) for h in got["predicted"]] == [len(h) for h in ref]


def test_one_beam_is_the_greedy_decode(ctx2):
    prefix = _prefix(40, 3)
    for steps in (1, 7, 8, 9, 30):
        got, greedy = ctx2.gpt_kv_beam(prefix, steps, 1), ctx2.gpt_kv_greedy(prefix, steps)
        assert got["predicted"][0].tolist() == greedy["predicted"].tolist()


def test_finished_hypotheses_stay_and_the_search_ends(mit2, tensors, gpt2_t):
    """With the stop token likely, hypotheses finish and keep their scores; the search ends before its steps do."""
    t = dict(gpt2_t)
    bias = t["gpt.mel_head.bias"].copy()
    bias[8193] += 4.0
    t["gpt.mel_head.bias"] = bias
    with mit2.Context({**tensors, **t}, device=0) as c:
        got = c.gpt_kv_beam(_prefix(10, 4), 400, 3)
        lens = [len(h) for h in got["predicted"]]
        print("lengths", lens, "scores", got["scores"], flush=True)
        assert all(h[-1] == 8193 and 8193 not in h[:-1] for h in got["predicted"]) and max(lens) < 400
        assert got["scores"].tolist() == sorted(got["scores"].tolist(), reverse=True)
        again = c.gpt_kv_beam(_prefix(10, 4), 399, 3)
        assert [h.tolist() for h in again["predicted"]] == [h.tolist() for h in got["predicted"]]
        assert again["scores"].tolist() == got["scores"].tolist()


def test_calls_of_changing_sizes_and_beside_greedy(ctx2):
    """Searches of other sizes before and greedy calls between do not show."""
    prefix = _prefix(70, 5)
    first = ctx2.gpt_kv_beam(prefix, 20, 3)
    greedy = ctx2.gpt_kv_greedy(prefix, 12)
    for P, steps, beams in ((3, 2, 8), (300, 40, 2), (0, 1, 1)):
        ctx2.gpt_kv_beam(_prefix(P, 9), steps, beams)
    again = ctx2.gpt_kv_beam(prefix, 20, 3)
    assert [h.tolist() for h in again["predicted"]] == [h.tolist() for h in first["predicted"]]
    assert again["scores"].tolist() == first["scores"].tolist()
    assert ctx2.gpt_kv_greedy(prefix, 12)["predicted"].tolist() == greedy["predicted"].tolist()


def test_a_search_that_does_not_fit_leaves_the_context_usable(mit2, ctx2):
    """With little GPU memory left, a long prefix's pages cannot be had: an error of the call; the next searches are as before."""
    torch = pytest.importorskip("torch")
    prefix = _prefix(40, 8)
    first = ctx2.gpt_kv_beam(prefix, 6, 3)
    free, _ = torch.cuda.mem_get_info()
    held = torch.empty(max(free - (3 << 30), 0), dtype=torch.uint8, device="cuda:0")
    try:
        with pytest.raises(mit2.Mit2CfmError) as e:
            ctx2.gpt_kv_beam(np.zeros((30000, 1280), np.float32), 6, 8)  # (its pages: 5 GB)
        assert e.value.status == mit2.E_HIP
        again = ctx2.gpt_kv_beam(prefix, 6, 3)
    finally:
        del held
        torch.cuda.empty_cache()
    assert [h.tolist() for h in again["predicted"]] == [h.tolist() for h in first["predicted"]]
    assert again["scores"].tolist() == first["scores"].tolist()


def test_refusals(mit2, ctx2, tensors):
    prefix = _prefix(2, 6)
    for steps, beams, hf in ((0, 3, False), (1819, 3, False), (1818, 3, True), (3, 0, False), (3, 9, False)):
        with pytest.raises(mit2.Mit2CfmError) as e:
            ctx2.gpt_kv_beam(prefix, steps, beams, hf)
        assert e.value.status == mit2.E_ARG
    with mit2.Context(tensors, device=0) as c, pytest.raises(mit2.Mit2CfmError) as e:
        c.gpt_kv_beam(prefix, 2)
    assert e.value.status == mit2.E_MODEL
