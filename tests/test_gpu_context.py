"""The operators for long and shared contexts as a decoder uses them together, on the GPU: steps of a batch whose sequences share
a prefix and whose caches are full (normed append, prefix attention, weights, eviction in all layers), eager and as a graph; two
contexts at once."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import context_ref  # noqa: E402
import ops_ref  # noqa: E402
from context_ref import DEV, check  # noqa: E402
from ops_ref import TORCH, Batch  # noqa: E402

pytestmark = pytest.mark.gpu
EPS, THETA, DECAY = 1e-6, 10000.0, 0.9


@pytest.fixture(scope="module")
def ctx(mit2):
    c = mit2.Context(synthetic_seed=3, device=0)
    yield c
    c.close()


class Decoder:
    """A batch's caches, accumulated weights and births in every layer, and one step's calls.  Sequences share their first rows'
    pages; each keeps `keep` rows, so that as many leave as come."""

    def __init__(self, mit2, *, layers=3, seqs=4, keep=150, shared=64, first=64, last=20, new=1, page=16, kv_heads=2, q_heads=4, dim=64, dtype="bf16", seed=0):
        self.mit2, self.layers, self.seqs, self.new, self.page, self.dtype = mit2, layers, seqs, new, page, dtype
        self.kv_heads, self.q_heads, self.dim, self.first, self.last, self.shared_rows, self.keep_rows = kv_heads, q_heads, dim, first, last, shared, keep
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        entries, full = -(-(keep + new) // page), shared // page
        pages = full + seqs * (entries - full)
        ids = rng.permutation(pages)
        table = np.empty((seqs, entries), np.int32)
        table[:, :full] = ids[:full]
        table[:, full:] = ids[full:].reshape(seqs, -1)
        t = TORCH[dtype]
        self.k, self.v = (torch.randn(layers, pages, kv_heads, page, dim, generator=g).to(t).to(DEV) for _ in range(2))
        self.table_np, self.pages, rows = table, pages, seqs * new
        self.table = torch.from_numpy(table).to(DEV)
        self.start = torch.arange(seqs + 1, dtype=torch.int32, device=DEV) * new
        self.length = torch.full((seqs,), keep, dtype=torch.int32, device=DEV)
        self.keep = torch.full((seqs,), keep, dtype=torch.int32, device=DEV)
        self.now = torch.tensor([keep + 10 * s for s in range(seqs)], dtype=torch.int32, device=DEV)  # (some have lost rows before)
        self.position = torch.zeros(rows, dtype=torch.int32, device=DEV)
        stride = entries * page
        self.weights = torch.rand(layers, seqs, kv_heads, stride, generator=g).to(DEV)
        self.born = torch.arange(stride, dtype=torch.int32).expand(layers, seqs, kv_heads, stride).contiguous().to(DEV)
        self.q, self.q_out, self.out = (torch.zeros(layers, rows, q_heads, dim, dtype=t, device=DEV) for _ in range(3))
        self.new_k, self.new_v = (torch.zeros(layers, rows, kv_heads, dim, dtype=t, device=DEV) for _ in range(2))
        self.q_weight, self.k_weight = ((1.0 + 0.2 * torch.randn(dim, generator=g)).to(t).to(DEV) for _ in range(2))
        self.lse = torch.zeros(layers, rows, q_heads, device=DEV)
        self.group = torch.tensor([0, seqs], dtype=torch.int32, device=DEV)
        self.shared = torch.tensor([shared], dtype=torch.int32, device=DEV)
        self.rng = torch.Generator(device=DEV).manual_seed(seed + 1)
        kw, qw = kv_heads * dim, q_heads * dim
        self.rows = mit2.KvRows(start=self.start.data_ptr(), length=self.length.data_ptr(), seqs=seqs, rows=rows, max_length=keep + new)
        self.norm = mit2.KvNorm(q_weight=self.q_weight.data_ptr(), k_weight=self.k_weight.data_ptr(), weight_dtype=mit2.DTYPES[dtype], eps=EPS)
        self.calls = []
        self.room = []
        for n in range(layers):
            cache = mit2.KvCache(k=self.k[n].data_ptr(), v=self.v[n].data_ptr(), table=self.table.data_ptr(), pages=pages, page_rows=page, kv_heads=kv_heads,
                                 head_dim=dim, table_stride=entries, dtype=mit2.DTYPES[dtype])
            put = mit2.KvAppend(k=self.new_k[n].data_ptr(), v=self.new_v[n].data_ptr(), k_row=kw, k_head=dim, v_row=kw, v_head=dim, q=self.q[n].data_ptr(),
                                q_out=self.q_out[n].data_ptr(), q_row=qw, q_head=dim, q_out_row=qw, q_out_head=dim, q_heads=q_heads,
                                position=self.position.data_ptr(), rotary_dim=dim, interleaved=0, theta=THETA)
            att = mit2.KvAttention(q=self.q_out[n].data_ptr(), out=self.out[n].data_ptr(), q_row=qw, q_head=dim, out_row=qw, out_head=dim, q_heads=q_heads,
                                   scale=dim ** -0.5)
            pre = mit2.KvPrefix(group=self.group.data_ptr(), shared=self.shared.data_ptr(), groups=1, max_shared=shared, lse=self.lse[n].data_ptr())
            size = mit2.kv_prefix_attention_workspace(cache, self.rows, q_heads, pre)
            self.room.append(torch.full((size,), 255, dtype=torch.uint8, device=DEV))
            att.workspace, att.workspace_bytes = self.room[-1].data_ptr(), size
            add = mit2.KvWeigh(q=self.q_out[n].data_ptr(), q_row=qw, q_head=dim, q_heads=q_heads, scale=dim ** -0.5, lse=self.lse[n].data_ptr(),
                               weights=self.weights[n].data_ptr(), weights_out=self.weights[n].data_ptr(), weight_stride=stride, decay=DECAY,
                               position=self.position.data_ptr(), born=self.born[n].data_ptr())
            self.calls.append((cache, put, att, pre, add))
        self.evict = mit2.KvEvict(seqs=seqs, layers=layers, layer_stride=self.k.stride(0), length=self.length.data_ptr(), keep=self.keep.data_ptr(),
                                  first_rows=first, last_rows=last, max_length=keep + new, weights=self.weights.data_ptr(),
                                  weights_out=self.weights.data_ptr(), weight_stride=stride, born=self.born.data_ptr(), born_out=self.born.data_ptr(),
                                  now=self.now.data_ptr(), length_out=self.length.data_ptr())
        size = mit2.kv_evict_workspace(self.calls[0][0], self.evict)
        self.room.append(torch.full((size,), 255, dtype=torch.uint8, device=DEV))
        self.evict.workspace, self.evict.workspace_bytes = self.room[-1].data_ptr(), size

    def arrive(self):
        """A step's new rows: projections, lengths with them, positions."""
        for x in (self.q, self.new_k, self.new_v):
            x.normal_(generator=self.rng)
        self.length += self.new
        self.position.copy_((self.now[:, None] + torch.arange(self.new, dtype=torch.int32, device=DEV)).reshape(-1))
        self.now += self.new
        torch.cuda.synchronize()

    def enqueue(self, ctx):
        for cache, put, att, pre, add in self.calls:
            ctx.kv_norm_append_device(cache, self.rows, put, self.norm)
            ctx.kv_prefix_attention_device(cache, self.rows, att, pre)
            ctx.kv_weigh_device(cache, self.rows, add)
        ctx.kv_evict_device(self.calls[0][0], self.evict)

    def batch(self, n):
        """Layer n as it is now, for the restatements."""
        b = Batch([self.new] * self.seqs, self.length.tolist(), page=self.page, kv_heads=self.kv_heads, q_heads=self.q_heads, dim=self.dim, dtype=self.dtype)
        b.table, b.pages = self.table_np, self.pages
        b.k, b.v, b.new_k, b.new_v = (x[n].cpu().clone() for x in (self.k, self.v, self.new_k, self.new_v))
        return b

    def tensors(self):
        return [self.k, self.v, self.q_out, self.out, self.lse, self.weights, self.born, self.length]


@pytest.mark.parametrize("dtype,dim,heads,new", [("f32", 64, (4, 4), 1), ("bf16", 128, (8, 2), 1), ("f16", 64, (4, 2), 5)])
def test_steps_of_full_caches(mit2, ctx, dtype, dim, heads, new):
    """Every call of a few steps against its restatement on the state that it met."""
    d = Decoder(mit2, q_heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, new=new, seed=dim)
    for step in range(3):
        d.arrive()
        position = d.position.cpu().numpy()
        for n, (cache, put, att, pre, add) in enumerate(d.calls):
            what = f"step {step} layer {n} {dtype}"
            b = d.batch(n)
            b.q = d.q[n].cpu()
            ctx.kv_norm_append_device(cache, d.rows, put, d.norm, sync=True)
            q, qt, k, kt, v = context_ref.norm_append64(b, d.q_weight.cpu()[None], d.k_weight.cpu()[None], d.norm.eps, False, position, dim, False, THETA)
            check(d.q_out[n].double().cpu(), q, qt, "q " + what)
            check(d.k[n].double().cpu(), k, kt, "k " + what)
            assert torch.equal(d.v[n].double().cpu(), v)
            b = d.batch(n)
            b.q = d.q_out[n].cpu()
            ctx.kv_prefix_attention_device(cache, d.rows, att, pre, sync=True)
            ref, tol = ops_ref.attention64(b, dim ** -0.5)
            check(d.out[n].double().cpu(), ref, tol, "out " + what)
            check(d.lse[n].double().cpu(), context_ref.lse64(b, dim ** -0.5), context_ref.lse_tolerance(b, dim ** -0.5), "lse " + what)
            before = d.weights[n].cpu()
            ctx.kv_weigh_device(cache, d.rows, add, sync=True)
            ref, tol = context_ref.weigh64(b, d.lse[n].cpu(), before, dim ** -0.5, decay=DECAY)
            check(d.weights[n].double().cpu(), ref, tol, "weights " + what)
        before = [x.cpu() for x in (d.k, d.v, d.weights, d.born)]
        lens = d.length.tolist()
        ctx.kv_evict_device(d.calls[0][0], d.evict, sync=True)
        k, v, w, births, left = context_ref.evict(before[0].double().numpy(), before[1].double().numpy(), d.table_np, d.page, lens, [d.keep_rows] * d.seqs,
                                                  before[2].numpy(), d.first, d.last, before[3].numpy(), d.now.tolist())
        assert d.length.tolist() == left.tolist() == [d.keep_rows] * d.seqs
        assert np.array_equal(d.k.double().cpu().numpy(), k) and np.array_equal(d.v.double().cpu().numpy(), v)
        assert np.array_equal(d.weights.cpu().numpy()[..., : d.keep_rows], w[..., : d.keep_rows])
        assert np.array_equal(d.born.cpu().numpy()[..., : d.keep_rows], births[..., : d.keep_rows])
        # the shared rows' pages are everybody's, and as they were
        shared = d.table_np[0, : d.shared_rows // d.page]
        assert torch.equal(d.k[:, shared].cpu(), before[0][:, shared])


class Graph:
    """The context's stream captured into a graph."""

    def __init__(self, ctx, enqueue):
        self.hip, self.stream = ctypes.CDLL("libamdhip64.so.7"), ctypes.c_void_p(ctx.stream)
        self.graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0  # hipStreamCaptureModeThreadLocal
        try:
            enqueue()
        finally:
            assert self.hip.hipStreamEndCapture(self.stream, ctypes.byref(self.graph)) == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exe), self.graph, None, None, ctypes.c_size_t(0)) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exe, self.stream) == 0
        assert self.hip.hipStreamSynchronize(self.stream) == 0

    def close(self):
        self.hip.hipGraphExecDestroy(self.exe)
        self.hip.hipGraphDestroy(self.graph)


@pytest.mark.parametrize("dtype,dim,new,keep", [("f32", 64, 1, 150), ("bf16", 128, 1, 300), ("f16", 64, 40, 200), ("bf16", 64, 1, 17000)])
def test_steps_as_a_graph(mit2, ctx, dtype, dim, new, keep):
    """A step captured once and replayed, with a twin's eager steps between the replays: the same to the bit.  (17000 rows: the
    eviction's lines in segments.)"""
    sizes = dict(dim=dim, dtype=dtype, new=new, keep=keep, seed=dim + new, layers=2)
    one, twin = Decoder(mit2, **sizes), Decoder(mit2, **sizes)
    torch.cuda.synchronize()
    g = Graph(ctx, lambda: one.enqueue(ctx))
    try:
        for step in range(5):
            for d in (one, twin):
                d.arrive()
            twin.enqueue(ctx)
            ctx.synchronize()
            g.replay()
            for a, b in zip(one.tensors(), twin.tensors()):
                assert torch.equal(a, b), (step, a.shape)
            assert bool(torch.isfinite(one.out.float()).all()) and one.length.tolist() == [keep] * one.seqs
    finally:
        g.close()


def test_two_contexts_at_once(mit2, ctx):
    """Two decoders on two contexts' streams, with workspaces of their own, step by step at the same time: as each alone."""
    other = mit2.Context(synthetic_seed=3, device=0)
    try:
        sizes = dict(dtype="bf16", dim=128, keep=700, shared=320, first=320, seqs=8, layers=4)
        both = [Decoder(mit2, seed=s, **sizes) for s in (1, 2)]
        alone = [Decoder(mit2, seed=s, **sizes) for s in (1, 2)]
        for d in alone:
            for _ in range(6):
                d.arrive()
                d.enqueue(ctx)
                ctx.synchronize()
        for _ in range(6):
            for d in both:
                d.arrive()
            for c, d in zip((ctx, other), both):
                d.enqueue(c)
            ctx.synchronize()
            other.synchronize()
        for d, e in zip(both, alone):
            for a, b in zip(d.tensors(), e.tensors()):
                assert torch.equal(a, b)
    finally:
        other.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_the_prefix_attention_and_the_plain_one_agree(mit2, ctx, dtype):
    """The same call with and without the sharing said, and kv_attention's: equal to rounding."""
    b = Batch([1, 3, 40], [300, 290, 310], page=16, q_heads=4, kv_heads=2, dim=64, dtype=dtype, seed=3)
    context_ref.share(b, [0, 3], [250], True)
    ref, tol = ops_ref.attention64(b, 0.125)
    on = context_ref.On(mit2, b)
    args = on.attention_args()
    size = mit2.kv_attention_workspace(on.cache, on.rows, b.q_heads)
    room = torch.empty(size + 16, dtype=torch.uint8, device=DEV)
    args.workspace, args.workspace_bytes = room.data_ptr(), size
    torch.cuda.synchronize()
    ctx.kv_attention_device(on.cache, on.rows, args, sync=True)
    plain = on.out.double().cpu()
    for groups in (0, 1):
        bounds, shared = torch.tensor([0, 3], dtype=torch.int32, device=DEV), torch.tensor([250], dtype=torch.int32, device=DEV)
        pre = mit2.KvPrefix(group=bounds.data_ptr() if groups else None, shared=shared.data_ptr() if groups else None, groups=groups, max_shared=250)
        size = mit2.kv_prefix_attention_workspace(on.cache, on.rows, b.q_heads, pre)
        room = torch.empty(size, dtype=torch.uint8, device=DEV)
        args.workspace, args.workspace_bytes = room.data_ptr(), size
        on.out.fill_(math.nan)
        torch.cuda.synchronize()
        ctx.kv_prefix_attention_device(on.cache, on.rows, args, pre, sync=True)
        check(on.out.double().cpu(), ref, tol, f"groups {groups}")
        check(on.out.double().cpu(), plain, 2 * tol, f"groups {groups} and the plain one")
