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
