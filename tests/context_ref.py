"""Plain 64-bit restatements of the operators for long and shared contexts (mit2cfm_kv_norm_append, mit2cfm_kv_prefix_attention,
mit2cfm_kv_weigh, mit2cfm_kv_evict), one loop a row, on the CPU; batches and buffers as in ops_ref.py."""
from __future__ import annotations

import math

import numpy as np
import torch

from ops_ref import HALF_STEP, TORCH, U, rotate64

DEV = "cuda:0"


class On:
    """A batch's buffers on the GPU and the library's descriptions of them."""

    def __init__(self, mit2, b):
        self.mit2, self.b = mit2, b
        self.k, self.v, self.q = b.k.to(DEV), b.v.to(DEV), b.q.to(DEV)
        self.new_k, self.new_v = b.new_k.to(DEV), b.new_v.to(DEV)
        self.table, self.start = torch.from_numpy(b.table).to(DEV), torch.from_numpy(b.start).to(DEV)
        self.length = torch.tensor(b.length, dtype=torch.int32, device=DEV)
        self.out = torch.full(b.q.shape, math.nan, dtype=TORCH[b.dtype], device=DEV)
        self.cache = mit2.KvCache(k=self.k.data_ptr(), v=self.v.data_ptr(), table=self.table.data_ptr(), pages=b.pages, page_rows=b.page,
                                  kv_heads=b.kv_heads, head_dim=b.dim, table_stride=b.table.shape[1], dtype=mit2.DTYPES[b.dtype])
        self.rows = mit2.KvRows(start=self.start.data_ptr(), length=self.length.data_ptr(), seqs=len(b.new), rows=b.rows,
                                max_length=max(b.length + [0]))

    def append_args(self, position=None, rot=0, interleaved=False, theta=10000.0):
        b, d = self.b, self.b.dim
        self.position = None if position is None else torch.as_tensor(position, dtype=torch.int32, device=DEV)
        return self.mit2.KvAppend(k=self.new_k.data_ptr(), v=self.new_v.data_ptr(), k_row=b.kv_heads * d, k_head=d, v_row=b.kv_heads * d, v_head=d,
                                  q=self.q.data_ptr(), q_out=self.out.data_ptr(), q_row=b.q_heads * d, q_head=d, q_out_row=b.q_heads * d, q_out_head=d,
                                  q_heads=b.q_heads, position=None if position is None else self.position.data_ptr(), rotary_dim=rot,
                                  interleaved=int(interleaved), theta=theta)

    def attention_args(self, scale=None, mask=None):
        b, d = self.b, self.b.dim
        self.mask = None if mask is None else torch.from_numpy(mask.view(np.int32)).to(DEV)
        return self.mit2.KvAttention(q=self.q.data_ptr(), out=self.out.data_ptr(), q_row=b.q_heads * d, q_head=d, out_row=b.q_heads * d, out_head=d,
                                     q_heads=b.q_heads, scale=d ** -0.5 if scale is None else scale,
                                     mask=None if mask is None else self.mask.data_ptr(), mask_words=0 if mask is None else mask.shape[1])


def mine(b):
    """Whether a row is a sequence's."""
    m = torch.zeros(b.rows, dtype=torch.bool)
    m[int(b.start[0]): int(b.start[-1])] = True
    return m


def check(got, ref, tol, what):
    off = (got - ref).abs()
    off[(got == ref) | (torch.isnan(got) & torch.isnan(ref))] = 0.0
    off = torch.nan_to_num(off, nan=math.inf)
    worst = float((off / tol.clamp_min(1e-300)).amax()) if off.numel() else 0.0
    print(f"{what}: worst {worst:.3f} of the tolerance", flush=True)
    assert bool((off <= tol).all()), what


# ------------------------------------------------------------------ normed append
def norm64(x, weight, eps, centered):
    """([heads][dim] normalised in float64, its error in fp32): x [heads][dim], weight [heads or 1][dim] or None.

    The mean of dim squares is off by dim + 1 roundings, its root and reciprocal by two more, the products with weight and mean
    by three: (dim / 2 + 8) U of the result.  A mean that is taken off is off by dim + 1 roundings of the largest element, and so is
    each difference; through the squares' mean that comes in again, in proportion to the result."""
    y = x.double()
    dim = y.shape[-1]
    c = y.mean(-1, keepdim=True) if centered else torch.zeros_like(y[..., :1])
    r = 1.0 / torch.sqrt(((y - c) ** 2).mean(-1, keepdim=True) + eps)
    z = (y - c) * r
    e = (dim / 2 + 8) * U * z.abs()
    if centered:
        e = e + (dim + 2) * U * y.abs().amax(-1, keepdim=True) * r * (1.0 + z.abs())
    w = torch.ones_like(z) if weight is None else weight.double().expand_as(z)
    return z * w, e * w.abs()


def norm_append64(b, q_weight, k_weight, eps, centered, position, rot, interleaved, theta):
    """(q_out, its tolerance, k, its tolerance, v) in float64; rows of no sequence give NaN in q_out."""
    q = torch.full(b.q.shape, math.nan, dtype=torch.float64)
    qt = torch.zeros_like(q)
    k, v = b.k.double(), b.v.double()
    kt = torch.zeros_like(k)
    for row, s, i, before in b.each_row():
        p = before + i if position is None else int(position[row])
        # the angle: fp32 half turns (pi U), its cosine and sine a few ulp; far out the fp64 product's error of the turns
        turn = math.pi * U + 6 * U + 0.16 * max(abs(p), 1) * 2.0 ** -52 * 8 * math.pi

        def one(x, weight):
            y, e = norm64(x, weight, eps, centered)
            top = y.abs().amax(-1, keepdim=True)
            z = rotate64(y, p, rot, interleaved, theta)
            t = 2 * e.amax(-1, keepdim=True) + (2 * top * turn if rot else 0.0)
            # the result's rounding; below f16's smallest normal, 2^-14, its steps are 2^-24 throughout
            return z, t + HALF_STEP[b.dtype] * (z.abs() + t) + (2.0 ** -25 if b.dtype == "f16" else 0.0)

        q[row], qt[row] = one(b.q[row], q_weight)
        page = b.page_of(s, before + i)
        if page >= 0:
            at = (before + i) % b.page
            k[page, :, at], kt[page, :, at] = one(b.new_k[row], k_weight)
            v[page, :, at] = b.new_v[row].double()
    return q, qt, k, kt, v


# ------------------------------------------------------------------ attention weights
def seen(b, row, s, i, before, mask):
    """Cached places that a new row sees: [(place, page, slot)]."""
    at = []
    for j in range(max(0, b.length[s])):
        n = j - before
        if n >= 0 and (n > i if mask is None else not (n < 32 * mask.shape[1] and mask[row, n // 32] >> np.uint32(n % 32) & 1)):
            continue
        page = b.page_of(s, j)
        if page >= 0:
            at.append((j, page, j % b.page))
    return at


def lse64(b, scale, mask=None):
    """log sum exp of each row's scores [rows][q_heads] in float64: -inf where it sees nothing, NaN for rows of no sequence."""
    out = torch.full(b.q.shape[:2], math.nan, dtype=torch.float64)
    group = b.q_heads // b.kv_heads
    for row, s, i, before in b.each_row():
        at = seen(b, row, s, i, before, mask)
        if not at:
            out[row] = -math.inf
            continue
        _, pages, slots = (torch.tensor(x) for x in zip(*at))
        for h in range(b.kv_heads):
            z = b.q[row, h * group: (h + 1) * group].double() @ b.k[pages, h, slots].double().t() * scale
            out[row, h * group: (h + 1) * group] = torch.logsumexp(z, -1)
    return out


def weigh64(b, lse, weights, scale, mask=None, decay=1.0, last=0):
    """(weights_out, its tolerance) in float64; lse [rows][q_heads] and weights [seqs][kv_heads][stride] fp32.

    An exponential's argument is off by the score's error (dim products and sums, the scale) and by the roundings of it and of lse
    in powers of two; its value by one more.  Then the fp32 sums over rows and query heads, and the product and sum with the old."""
    out, tol = weights.double().clone(), torch.zeros(weights.shape, dtype=torch.float64)
    stride, group = weights.shape[2], b.q_heads // b.kv_heads
    decay = float(np.float32(decay))
    for s, n in enumerate(b.new):
        if n == 0:
            continue
        first = b.length[s] - n
        places = min(b.length[s], stride, b.table.shape[1] * b.page)
        for j in range(max(0, places)):
            out[s, :, j] = out[s, :, j] * decay if j < first else 0.0
        tol[s] = 3 * U * out[s].abs()
        tol[s, :, max(0, places):] = 0.0
    for row, s, i, before in b.each_row():
        if last and i < b.new[s] - last:
            continue
        at = [x for x in seen(b, row, s, i, before, mask) if x[0] < stride]
        if not at:
            continue
        places, pages, slots = (torch.tensor(x) for x in zip(*at))
        for h in range(b.kv_heads):
            k = b.k[pages, h, slots].double()
            q = b.q[row, h * group: (h + 1) * group].double()
            z, l = q @ k.t() * scale, lse[row, h * group: (h + 1) * group].double()[:, None]
            p = torch.where(l == -math.inf, 0.0, torch.exp(z - l))
            rel = (b.dim + 4) * U * abs(scale) * (q.abs() @ k.abs().t()) + 4 * U * (z.abs() + l.abs().nan_to_num(posinf=0.0)) + 8 * U
            out[s, h, places] += p.sum(0)
            tol[s, h, places] += (p * 1.01 * (rel + (b.new[s] * group + 8) * U)).sum(0) + group * 2.0 ** -120
    return out, tol


# ------------------------------------------------------------------ eviction
def evict(k, v, table, page, length, keep, weights, first, last, born=None, now=None):
    """kv_evict on numpy arrays: k, v [layers][pages][heads][page][dim], table [seqs][entries], weights and born
    [layers][seqs][heads][stride].  Returns (k, v, weights, born, length): places past the new lengths are NaN (-1) in the copies."""
    old_k, old_v, k, v = k, v, k.copy(), v.copy()
    pages = k.shape[1]
    new_w = np.full(weights.shape, np.nan, np.float32)
    new_b = None if born is None else np.full(born.shape, -1, np.int32)
    out = []
    for s in range(table.shape[0]):
        n = max(0, min(length[s], table.shape[1] * page, weights.shape[3]))
        m = min(n, max(0, keep[s]))
        out.append(m)
        for layer in range(weights.shape[0]):
            for h in range(weights.shape[2]):
                w = weights[layer, s, h, :n]
                rank = []
                for j in range(n):
                    stays = j < first or (j >= n - last if born is None else int(born[layer, s, h, j]) >= int(now[s]) - last)
                    least = np.isnan(w[j]) or not 0 <= table[s, j // page] < pages
                    rank.append((-2 if stays else 0 if least else -1, 0.0 if stays or least else -float(w[j]), j))
                kept = sorted(x[2] for x in sorted(rank)[:m])
                place = {j: j for j in kept if j < m}
                free = [j for j in range(m) if j not in place]
                for dst, src in zip(free, [j for j in kept if j >= m]):
                    place[dst] = src
                    a, b = int(table[s, src // page]), int(table[s, dst // page])
                    if 0 <= a < pages and 0 <= b < pages:
                        k[layer, b, h, dst % page], v[layer, b, h, dst % page] = old_k[layer, a, h, src % page], old_v[layer, a, h, src % page]
                for dst, src in place.items():
                    new_w[layer, s, h, dst] = w[src]
                    if born is not None:
                        new_b[layer, s, h, dst] = born[layer, s, h, src]
    return k, v, new_w, new_b, np.array(out, np.int32)


# ------------------------------------------------------------------ shared prefixes
def share(b, bounds, shared, alias):
    """Makes the first shared[g] rows of the sequences bounds[g] .. bounds[g + 1] - 1 of a batch alike: full pages by name when
    `alias`, else (and the last part page) by copies."""
    for g, n in enumerate(shared):
        lo, hi = bounds[g], bounds[g + 1]
        for s in range(lo + 1, hi):
            for j in range(min(n, b.length[s], b.length[lo])):
                if alias and (j // b.page + 1) * b.page <= n:
                    b.table[s, j // b.page] = b.table[lo, j // b.page]
                    continue
                frm, to, at = b.page_of(lo, j), b.page_of(s, j), j % b.page
                for x in (b.k, b.v):
                    x[to, :, at] = x[frm, :, at]


def lse_tolerance(b, scale, mask=None):
    """How far a log sum may be off: its scores' errors, weighted (dim products and sums, the scale, the exponentials), the sum's,
    and the maximum's and logarithm's roundings in powers of two."""
    tol = torch.zeros(b.q.shape[:2], dtype=torch.float64)
    group = b.q_heads // b.kv_heads
    for row, s, i, before in b.each_row():
        at = seen(b, row, s, i, before, mask)
        if not at:
            continue
        _, pages, slots = (torch.tensor(x) for x in zip(*at))
        for h in range(b.kv_heads):
            k, q = b.k[pages, h, slots].double(), b.q[row, h * group: (h + 1) * group].double()
            z = q @ k.t() * scale
            score = (b.dim + 4) * U * abs(scale) * (q.abs() @ k.abs().t()) + 4 * U * z.abs() + 4 * U
            lse = torch.logsumexp(z, -1)
            tol[row, h * group: (h + 1) * group] = 1.01 * (torch.softmax(z, -1) * score).sum(-1) + (len(at) + 16) * U + 6 * U * lse.abs()
    return tol
