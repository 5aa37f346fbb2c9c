"""Plain 64-bit restatements of the paged-cache and beam operators (mit2cfm_kv_*,
mit2cfm_beam_*), one loop a row, on the CPU; and what a test batch is made of."""
from __future__ import annotations

import math

import numpy as np
import torch

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {k: torch.finfo(t).eps / 2 for k, t in TORCH.items()}  # a rounding's largest relative error
U = 2.0 ** -24  # fp32's


class Batch:
    """A paged cache on the CPU with ragged sequences: new[s] new rows, length[s] cached rows with them."""

    def __init__(self, new, length, *, page=16, kv_heads=2, q_heads=4, dim=64, dtype="f32", seed=0, spare=3, tail_rows=0,
                 lead_rows=0, extra_entries=1):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.new, self.length, self.page, self.dtype = list(new), list(length), page, dtype
        self.kv_heads, self.q_heads, self.dim = kv_heads, q_heads, dim
        held = [-(-n // page) for n in length]
        self.pages = sum(held) + spare
        ids = rng.permutation(self.pages)
        self.table = np.full((len(new), max(held + [0]) + extra_entries), -1, np.int32)
        at = 0
        for s, n in enumerate(held):
            self.table[s, :n] = ids[at: at + n]
            at += n
        self.start = np.concatenate([[lead_rows], lead_rows + np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.start[-1]) + tail_rows

        def normal(*shape):
            return torch.randn(*shape, generator=g).to(TORCH[dtype])

        self.k, self.v = (normal(self.pages, kv_heads, page, dim) for _ in range(2))
        self.q = normal(self.rows, q_heads, dim)
        self.new_k, self.new_v = (normal(self.rows, kv_heads, dim) for _ in range(2))

    def each_row(self):
        """(row, sequence, index among its new rows, cached rows before the new ones)."""
        for s, n in enumerate(self.new):
            for i in range(n):
                yield int(self.start[s]) + i, s, i, self.length[s] - n

    def page_of(self, s, j):
        if not 0 <= j < self.table.shape[1] * self.page:
            return -1
        p = int(self.table[s, j // self.page])
        return p if 0 <= p < self.pages else -1


def rotate64(x, position, rot, interleaved, theta):
    """x [heads][dim] in float64, its first rot elements turned."""
    y = x.double().clone()
    half = rot // 2
    a = position * theta ** (-2.0 * torch.arange(half, dtype=torch.float64) / max(rot, 1))
    cos, sin = torch.cos(a), torch.sin(a)
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, half), slice(half, rot))
    u, w = x[:, lo].double(), x[:, hi].double()
    y[:, lo], y[:, hi] = u * cos - w * sin, w * cos + u * sin
    return y


def append64(b: Batch, position, rot, interleaved, theta):
    """(q_out, k, v) in float64; rows of no sequence give NaN in q_out (nothing is written there)."""
    q = torch.full(b.q.shape, math.nan, dtype=torch.float64)
    k, v = b.k.double(), b.v.double()
    for row, s, i, before in b.each_row():
        p = before + i if position is None else int(position[row])
        q[row] = rotate64(b.q[row], p, rot, interleaved, theta)
        page = b.page_of(s, before + i)
        if page >= 0:
            k[page, :, (before + i) % b.page] = rotate64(b.new_k[row], p, rot, interleaved, theta)
            v[page, :, (before + i) % b.page] = b.new_v[row].double()
    return q, k, v


def visible(b: Batch, row, s, i, before, mask):
    """Cached rows that a new row sees: [(page, slot)]."""
    at = []
    for j in range(max(0, b.length[s])):
        n = j - before
        if n >= 0 and (n > i if mask is None else not (n < 32 * mask.shape[1] and mask[row, n // 32] >> np.uint32(n % 32) & 1)):
            continue
        page = b.page_of(s, j)
        if page >= 0:
            at.append((page, j % b.page))
    return at


def attention64(b: Batch, scale, mask=None):
    """(out, tolerance) in float64.  The tolerance counts, for each row and head: a score's error (its dim products and sums and
    the scale in fp32, its exponential's argument and value), the fp32 sums over the keys, and with 16-bit types the
    probabilities' rounding and the result's."""
    out = torch.full(b.q.shape, math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    group = b.q_heads // b.kv_heads
    for row, s, i, before in b.each_row():
        at = visible(b, row, s, i, before, mask)
        if not at:
            out[row] = 0.0
            continue
        pages, slots = (torch.tensor(x) for x in zip(*at))
        for h in range(b.kv_heads):
            k, v = b.k[pages, h, slots].double(), b.v[pages, h, slots].double()
            q = b.q[row, h * group: (h + 1) * group].double()
            z = q @ k.t() * scale
            p = torch.softmax(z, -1)
            o = p @ v
            # each score's error; a probability is off by it and by the mean of all (to first order: 1.01 covers the rest)
            score = (b.dim + 4) * U * abs(scale) * (q.abs() @ k.abs().t()) + 4 * U * z.abs() + 4 * U
            spread = p @ v.abs()
            e = 1.01 * ((p * score) @ v.abs() + (p * score).sum(-1, keepdim=True) * o.abs()) + (len(at) + 16) * U * (spread + o.abs())
            if b.dtype != "f32":
                e = e + HALF_STEP[b.dtype] * spread
            out[row, h * group: (h + 1) * group] = o
            tol[row, h * group: (h + 1) * group] = e + HALF_STEP[b.dtype] * (o.abs() + e)
    return out, tol


def bits(sees):
    """A mask's words [rows][words] from whether row i sees new row j [rows][n]."""
    rows, n = sees.shape
    wide = np.zeros((rows, -(-n // 32) * 32), bool)
    wide[:, :n] = sees
    return np.packbits(wide, axis=1, bitorder="little").view(np.uint32)


def trees(b: Batch, seed, words=None):
    """A random tree's mask over every sequence's new rows, and the rows' depths."""
    rng = np.random.default_rng(seed)
    most = max(b.new + [1])
    sees, depth = np.zeros((b.rows, most), bool), np.zeros(b.rows, np.int32)
    for row, s, i, _ in b.each_row():
        parent = int(rng.integers(-1, i)) if i else -1
        if parent >= 0:
            sees[row] = sees[b.start[s] + parent]
            depth[row] = depth[b.start[s] + parent] + 1
        sees[row, i] = True
    return bits(sees), depth


def select64(logits, scores, count, finished=None, stop=-1):
    """(scores, parents, tokens, finished) of beam_select: logits [groups][beams][vocab] float64, scores [groups][beams]."""
    groups, beams, vocab = logits.shape
    res = [np.empty((groups, count), t) for t in (np.float64, np.int32, np.int32, np.int32)]
    for g in range(groups):
        flat = np.full((beams, vocab), -np.inf)
        for b in range(beams):
            c = scores[g, b]
            if not c > -np.inf:
                continue
            if finished is not None and finished[g, b]:
                flat[b, stop] = c
                continue
            x = np.where(np.isnan(logits[g, b]), -np.inf, np.minimum(logits[g, b], np.finfo(np.float32).max))
            m = x.max()
            if m > -np.inf:
                flat[b] = c + (x - (m + math.log(np.exp(x - m).sum())))
        order = np.lexsort((np.arange(beams * vocab), -flat.reshape(-1)))[:count]
        res[0][g], res[1][g], res[2][g] = flat.reshape(-1)[order], order // vocab, order % vocab
        res[3][g] = (res[2][g] == stop) | (finished[g][res[1][g]] != 0 if finished is not None else False)
    return res


def owners(parent):
    """For one group's parents: whose full pages each new beam has, whose private pages, and whether it is a further child."""
    beams = len(parent)
    parent = [p if 0 <= p < beams else r for r, p in enumerate(parent)]
    bare = [r for r in range(beams) if r not in parent]
    owner, further = [], []
    for r, p in enumerate(parent):
        again = p in parent[:r]
        further.append(again)
        owner.append(bare.pop(0) if again else p)
    return parent, owner, further


def reorder(k, v, table, page, parent, length, state=None, token=None, place=None):
    """beam_reorder on numpy arrays: k, v [layers][pages][heads][page][dim], table [groups][beams][entries], state [groups][beams][words]."""
    k, v = k.copy(), v.copy()
    old_k, old_v = k.copy(), v.copy()
    out = np.empty_like(table)
    new_state = None if state is None else np.empty_like(state)
    pages = k.shape[1]
    for g in range(table.shape[0]):
        p, owner, further = owners(list(parent[g][: table.shape[1]]))
        n = length[g] if 0 <= length[g] <= table.shape[2] * page else table.shape[2] * page
        full, part = n // page, n % page
        for r in range(table.shape[1]):
            out[g, r, :full] = table[g, p[r], :full]
            out[g, r, full:] = table[g, owner[r], full:]
            if further[r] and part:
                frm, to = table[g, p[r], full], table[g, owner[r], full]
                if 0 <= frm < pages and 0 <= to < pages:
                    k[:, to, :, :part], v[:, to, :, :part] = old_k[:, frm, :, :part], old_v[:, frm, :, :part]
            if state is not None:
                new_state[g, r] = state[g, p[r]]
                if token is not None and 0 <= place[g] < state.shape[2]:
                    new_state[g, r, place[g]] = token[g, r]
    return out, k, v, new_state
