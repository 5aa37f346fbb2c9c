"""The operators over a paged key/value cache and a beam search's states, as a decoding program calls them.

Each case is one call through the Python binding (`mit2cfm.Context`), on buffers that lie on the GPU:

  append     kv_append_device: new rows' keys (rotated) and values into a paged cache, their queries rotated
  attention  kv_attention_device: new rows' attention over the cache: single tokens, chains, trees of drafted tokens
  select     beam_select_device: a step's best continuations over beams and vocabulary
  reorder    beam_reorder_device: page tables, the last part page and the states after a selection

Sizes are the GPT decoder's (20 heads of 64, 8194 codes, 24 layers), the estimator's (8 heads of 64) or generic
ones (32 query heads on 8 key heads of 128); `draw` spreads over the same ranges.  The plain forms are elementary
torch operations; `exact` restates each operator in float64 from its definition.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False  # True: `run` calls the library, False: the plain forms

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 10000.0


# ------------------------------------------------------------------ the cases
def listed():
    gpt = dict(q_heads=20, kv_heads=20, dim=64, dtype="f32", page=64)
    wide = dict(q_heads=32, kv_heads=8, dim=128, dtype="bf16")
    return [
        # one step of a three-beam search with the GPT decoder's heads: the smallest call
        dict(name="append_step_3", kind="append", seqs=3, new=1, length=703, ragged=False, tree=False, rot=0, interleaved=False, **gpt),
        # drafted trees of a batch, each token at its depth's position
        dict(name="append_tree_16", kind="append", seqs=16, new=25, length=1700, ragged=True, tree=True, rot=128, interleaved=False, page=16, **wide),
        # prompts of a batch in one call, lengths as they come
        dict(name="append_prompts_9", kind="append", seqs=9, new=2047, length=2900, ragged=True, tree=False, rot=64, interleaved=True, page=32, **wide),
        # the beams' step over their caches, fp32 as the GPT decoder keeps it
        dict(name="attend_step_3", kind="attention", seqs=3, new=1, length=703, ragged=False, tree=False, **gpt),
        # a serving batch, one token each, lengths as they come
        dict(name="attend_batch_64", kind="attention", seqs=64, new=1, length=8191, ragged=True, tree=False, page=16, **wide),
        # one long context: the split over the keys
        dict(name="attend_long_1", kind="attention", seqs=1, new=1, length=131001, ragged=False, tree=False, page=64, **wide),
        # drafted trees checked against the cache
        dict(name="attend_tree_8", kind="attention", seqs=8, new=63, length=4099, ragged=True, tree=True, page=32, **dict(wide, dtype="f16")),
        # a further piece of a prefix, fp32, each row seeing those before it
        dict(name="attend_chain_2", kind="attention", seqs=2, new=257, length=1201, ragged=True, tree=False, **gpt),
        # three beams over the mel codes
        dict(name="select_3", kind="select", groups=1, beams=3, vocab=8194, count=6, dtype="f32", finished=False),
        # a batch of searches over a large vocabulary, some hypotheses finished
        dict(name="select_32x8", kind="select", groups=32, beams=8, vocab=50001, count=16, dtype="bf16", finished=True),
        # three beams of the GPT decoder: 24 layers of pages, code histories
        dict(name="reorder_3", kind="reorder", groups=1, beams=3, prefix=150, length=653, layers=24, kv_heads=20, dim=64, page=64, dtype="f32", words=1819),
        # a batch of searches
        dict(name="reorder_32x8", kind="reorder", groups=32, beams=8, prefix=500, length=1021, layers=24, kv_heads=8, dim=64, page=32, dtype="bf16", words=513),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "append", "attention", "attention", "attention", "select", "reorder"])
    if kind == "select":
        return dict(kind=kind, groups=log(1, 31), beams=rng.randint(1, 8), vocab=log(100, 49999), count=rng.randint(1, 16),
                    dtype=rng.choice(["f32", "f16", "bf16"]), finished=rng.random() < 0.5)
    heads = rng.choice([(20, 20, 64), (8, 8, 64), (32, 8, 128), (24, 4, 96), (16, 2, 128), (7, 1, 32)])
    dtype, page = rng.choice(["f32", "f16", "bf16"]), rng.choice([8, 16, 32, 64, 128])
    if kind == "reorder":
        prefix = log(1, 600)
        groups = log(1, 30)
        return dict(kind=kind, groups=groups, beams=rng.randint(2, 8), prefix=prefix, length=prefix + log(1, 500),
                    layers=rng.randint(1, min(24, max(1, 160 // groups))), kv_heads=heads[1], dim=heads[2], page=min(page, 64),
                    dtype=dtype if heads[1] * heads[2] <= 512 else "f16", words=log(1, 1800))
    form = dict(q_heads=heads[0], kv_heads=heads[1], dim=heads[2], dtype=dtype, page=page)
    if kind == "append":
        seqs, tree = log(1, 64), rng.random() < 0.5
        new = rng.randint(2, 64) if tree else log(1, max(2, 6000 // seqs))
        rot = 2 * rng.randint(0, heads[2] // 2)
        return dict(kind=kind, seqs=seqs, new=new, length=new + log(1, 2000), ragged=rng.random() < 0.7, tree=tree, rot=rot,
                    interleaved=rng.random() < 0.5, **form)
    shape = rng.choice(["step", "step", "tree", "chain"])
    if shape == "step":
        seqs = log(1, 64)
        length = log(1, min(100000, 180000 // seqs))
        return dict(kind=kind, seqs=seqs, new=1, length=length, ragged=rng.random() < 0.7, tree=False, **form)
    seqs = log(1, 7)
    new = rng.randint(2, 100 if shape == "tree" else 250)
    return dict(kind=kind, seqs=seqs, new=new, length=new + log(1, 2500), ragged=rng.random() < 0.7, tree=shape == "tree", **form)


# ------------------------------------------------------------------ inputs
def _lens(case):
    """(new rows, cached rows with them) of each sequence; a ragged batch's first is the largest."""
    n = case["seqs"]
    u = [((5 * s) % n) / n if case["ragged"] else 0.0 for s in range(n)]
    new = [1 + int((case["new"] - 1) * (1.0 - 0.6 * x)) for x in u]
    return new, [max(k, round(case["length"] * (1.0 - 0.6 * x))) for k, x in zip(new, u)]


def _group_lens(case):
    """Cached rows of each group's beams."""
    return [case["length"] - (7 * g) % (case["length"] - case["prefix"]) for g in range(case["groups"])]


def _trees(seqs, new, rng):
    """Random trees over each sequence's new rows: whether row i's path from the root holds row j, and row i's depth."""
    n = max(new)
    sees = np.zeros((seqs, n, n), bool)
    depth = np.zeros((seqs, n), np.int64)
    every = np.arange(seqs)
    for i in range(n):
        parent = rng.integers(max(-1, i - 6), i, seqs) if i else np.full(seqs, -1)
        has = parent >= 0
        sees[has, i] = sees[every[has], parent[has]]
        depth[has, i] = depth[every[has], parent[has]] + 1
        sees[:, i, i] = True
    return sees, depth


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _inputs(case, seed):
    """Inputs from the seed alone."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, dtype = case["kind"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    if kind == "select":
        n, b, v = case["groups"], case["beams"], case["vocab"]
        d = dict(logits=normal(n, b, v) * 2.5, scores=-5.0 * torch.rand(n, b, generator=g, device=DEV), finished=None, stop=v - 1)
        if case["finished"]:
            d["finished"] = _ints(rng.random((n, b)) < 0.2)
        return d
    if kind == "reorder":
        n, b, page = case["groups"], case["beams"], case["page"]
        shared, most = case["prefix"] // page, -(-(case["length"] + 1) // page)
        pages = n * (shared + b * (most - shared))
        ids = rng.permutation(pages)
        table = np.empty((n, b, most), np.int64)
        table[:, :, :shared] = ids[: n * shared].reshape(n, 1, shared)
        table[:, :, shared:] = ids[n * shared:].reshape(n, b, most - shared)
        shape = (case["layers"], pages, case["kv_heads"], page, case["dim"])
        lens = np.array(_group_lens(case))
        return dict(k=normal(*shape), v=normal(*shape), table=_ints(table), parent=_ints(rng.integers(0, b, (n, b))), length=_ints(lens),
                    state=_ints(rng.integers(0, 8194, (n, b, case["words"]))), token=_ints(rng.integers(0, 8194, (n, b))),
                    place=_ints(np.minimum(lens - case["prefix"], case["words"] - 1)))
    new, lens = _lens(case)
    page, seqs, rows = case["page"], case["seqs"], sum(new)
    most = -(-max(lens) // page)
    held = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(held))
    table = np.zeros((seqs, most), np.int64)
    for s, at in enumerate(np.cumsum([0] + held[:-1])):
        table[s, : held[s]] = ids[at: at + held[s]]
    start = np.cumsum([0] + new)
    d = dict(table=_ints(table), start=_ints(start), length=_ints(lens), q=normal(rows, case["q_heads"], case["dim"]), mask=None, position=None,
             cache_k=normal(sum(held), case["kv_heads"], page, case["dim"]), cache_v=normal(sum(held), case["kv_heads"], page, case["dim"]))
    sees = None
    if case["tree"]:
        sees, depth = _trees(seqs, new, rng)
    if kind == "append":
        d.update(k=normal(rows, case["kv_heads"], case["dim"]), v=normal(rows, case["kv_heads"], case["dim"]))
        if case["tree"]:
            d["position"] = _ints(np.concatenate([lens[s] - new[s] + depth[s, : new[s]] for s in range(seqs)]))
    elif case["tree"]:
        words = -(-max(new) // 32)
        bits = np.zeros((rows, words * 32), bool)
        for s in range(seqs):
            bits[start[s]: start[s + 1], : new[s]] = sees[s, : new[s], : new[s]]
        d["mask"] = _ints(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
    return d


_shared: dict = {}


def _binding():
    """The library's Python binding and this process's context."""
    if not _shared:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "index-tts2-metal_amd"))
        import mit2cfm

        _shared.update(mit2cfm=mit2cfm, ctx=mit2cfm.Context(synthetic_seed=1, device=0))
    return _shared["mit2cfm"], _shared["ctx"]


def _plan(s):
    """The library's descriptions of a state's buffers, and its workspace."""
    mit2cfm, s["ctx"] = _binding()
    case, kind = s["case"], s["case"]["kind"]

    def at(name):
        return s[name].data_ptr() if s.get(name) is not None else None

    if kind == "select":
        a = mit2cfm.BeamSelect(logits=at("logits"), logits_row=case["vocab"], dtype=mit2cfm.DTYPES[case["dtype"]], groups=case["groups"],
                               beams=case["beams"], vocab=case["vocab"], count=case["count"], scores=at("scores"), finished=at("finished"),
                               stop_token=s["stop"], scores_out=at("scores_out"), parent_out=at("parent_out"), token_out=at("token_out"),
                               finished_out=at("finished_out"))
        s["workspace"] = torch.empty(max(16, mit2cfm.beam_select_workspace(a)), dtype=torch.uint8, device=DEV)
        a.workspace, a.workspace_bytes = at("workspace"), s["workspace"].numel()
        return dict(args=a)
    if kind == "reorder":
        cache = mit2cfm.KvCache(k=at("k"), v=at("v"), table=at("table"), pages=s["k"].shape[1], page_rows=case["page"], kv_heads=case["kv_heads"],
                                head_dim=case["dim"], table_stride=s["table"].shape[-1], dtype=mit2cfm.DTYPES[case["dtype"]])
        a = mit2cfm.BeamReorder(groups=case["groups"], beams=case["beams"], layers=case["layers"], layer_stride=s["k"].stride(0), parent=at("parent"),
                                parent_stride=case["beams"], length=at("length"), table_out=at("table_out"), state=at("state"),
                                state_out=at("state_out"), state_words=case["words"], token=at("token"), place=at("place"))
        return dict(cache=cache, args=a)
    cache = mit2cfm.KvCache(k=at("cache_k"), v=at("cache_v"), table=at("table"), pages=s["cache_k"].shape[0], page_rows=case["page"],
                            kv_heads=case["kv_heads"], head_dim=case["dim"], table_stride=s["table"].shape[1], dtype=mit2cfm.DTYPES[case["dtype"]])
    new, lens = _lens(case)
    rows = mit2cfm.KvRows(start=at("start"), length=at("length"), seqs=case["seqs"], rows=sum(new), max_length=max(lens))
    d, qw, kw = case["dim"], case["dim"] * case["q_heads"], case["dim"] * case["kv_heads"]
    if kind == "append":
        a = mit2cfm.KvAppend(k=at("k"), v=at("v"), k_row=kw, k_head=d, v_row=kw, v_head=d, q=at("q"), q_out=at("out"), q_row=qw, q_head=d,
                             q_out_row=qw, q_out_head=d, q_heads=case["q_heads"], position=at("position"), rotary_dim=case["rot"],
                             interleaved=int(case["interleaved"]), theta=THETA)
    else:
        a = mit2cfm.KvAttention(q=at("q"), out=at("out"), q_row=qw, q_head=d, out_row=qw, out_head=d, q_heads=case["q_heads"],
                                scale=1.0 / math.sqrt(d), mask=at("mask"), mask_words=0 if s["mask"] is None else s["mask"].shape[1])
        s["workspace"] = torch.empty(max(16, mit2cfm.kv_attention_workspace(cache, rows, case["q_heads"])), dtype=torch.uint8, device=DEV)
        a.workspace, a.workspace_bytes = at("workspace"), s["workspace"].numel()
    return dict(cache=cache, rows=rows, args=a)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind == "select":
        n, c = case["groups"], case["count"]
        s["scores_out"] = torch.empty(n, c, device=DEV)
        for name in ("parent_out", "token_out", "finished_out"):
            s[name] = torch.empty(n, c, dtype=torch.int32, device=DEV)
    elif kind == "reorder":
        s["table_out"], s["state_out"] = torch.empty_like(s["table"]), torch.empty_like(s["state"])
    else:
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["plan"] = _plan(s)
    torch.cuda.synchronize()  # a context works on a stream of its own
    return s


# ------------------------------------------------------------------ one pass
def _outputs(s):
    kind = s["case"]["kind"]
    if kind == "append":
        return {"q": s["out"], "k": s["cache_k"], "v": s["cache_v"]}
    if kind == "attention":
        return s["out"]
    if kind == "select":
        return {"scores": s["scores_out"], "parent": s["parent_out"], "token": s["token_out"], "finished": s["finished_out"]}
    return {"table": s["table_out"], "state": s["state_out"], "k": s["k"], "v": s["v"]}


def run(s):
    kind = s["case"]["kind"]
    if own:
        p = s["plan"]
        if kind == "append":
            s["ctx"].kv_append_device(p["cache"], p["rows"], p["args"])
        elif kind == "attention":
            s["ctx"].kv_attention_device(p["cache"], p["rows"], p["args"])
        elif kind == "select":
            s["ctx"].beam_select_device(p["args"])
        else:
            s["ctx"].beam_reorder_device(p["cache"], p["args"])
        return _outputs(s)
    {"append": _append, "attention": _attention, "select": _select, "reorder": _reorder}[kind](s)
    return _outputs(s)


# ------------------------------------------------------------------ plain forms
def _places(s):
    """Each new row's sequence and its place there."""
    start, length = s["start"].long(), s["length"].long()
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(start[1:], row, right=True)
    return seq, row - start[seq], length[seq] - (start[seq + 1] - start[seq])


def _rotated(x, position, case):
    half = case["rot"] // 2
    if half == 0:
        return x
    # far positions: the angle in 64 bits
    a = position.double()[:, None] * torch.exp(torch.arange(half, device=DEV).double() * (-2.0 * math.log(THETA) / case["rot"]))
    cos, sin = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    y = x.float()
    r, rest = y[..., : case["rot"]], y[..., case["rot"]:]
    if case["interleaved"]:
        u, w = r[..., 0::2], r[..., 1::2]
        r = torch.stack([u * cos - w * sin, w * cos + u * sin], -1).flatten(-2)
    else:
        u, w = r[..., :half], r[..., half:]
        r = torch.cat([u * cos - w * sin, w * cos + u * sin], -1)
    return torch.cat([r, rest], -1).to(x.dtype)


def _append(s):
    case = s["case"]
    seq, i, before = _places(s)
    place = before + i
    position = place if s["position"] is None else s["position"]
    page = s["table"].long()[seq, place // case["page"]]
    s["cache_k"][page, :, place % case["page"]] = _rotated(s["k"], position, case)
    s["cache_v"][page, :, place % case["page"]] = s["v"]
    s["out"].copy_(_rotated(s["q"], position, case))


def _attention(s):
    case = s["case"]
    seqs, kvh, d, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    group, new = case["q_heads"] // kvh, case["new"]
    seq, i, before = _places(s)
    start = s["start"].long()

    def rows_of(cache):  # [seqs][kv heads][cached rows][dim]
        return cache[s["table"].long()].transpose(1, 2).reshape(seqs, kvh, -1, d).float()

    k, v = rows_of(s["cache_k"]), rows_of(s["cache_v"])
    n = k.shape[2]
    q = torch.zeros(seqs, new, kvh, group, d, device=DEV)
    q[seq, i] = s["q"].float().view(-1, kvh, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * new, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    # which keys a row sees: those before the new rows, and of the new rows its path (a chain: those up to itself)
    first = (s["length"].long() - (start[1:] - start[:-1]))[:, None]
    j = torch.arange(n, device=DEV)[None] - first
    if s["mask"] is None:
        sees = j[:, None] <= torch.arange(new, device=DEV)[None, :, None]
    else:
        bits = torch.zeros(seqs, new, s["mask"].shape[1], dtype=torch.int32, device=DEV)
        bits[seq, i] = s["mask"]
        on = (bits[..., None] >> torch.arange(32, dtype=torch.int32, device=DEV)) & 1
        on = on.flatten(2).bool()
        sees = torch.gather(on, 2, j.clamp(0, on.shape[2] - 1)[:, None].expand(seqs, new, n)) & (j < on.shape[2])[:, None] | (j < 0)[:, None]
    sees = sees & (torch.arange(n, device=DEV)[None, None] < s["length"].long()[:, None, None])
    sees = sees[:, None, None].expand(seqs, kvh, group, new, n).reshape(seqs, kvh, group * new, n)
    score = score.masked_fill(~sees, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = out.view(seqs, kvh, group, new, d).permute(0, 3, 1, 2, 4).reshape(seqs, new, case["q_heads"], d)
    s["out"].copy_(out[seq, i].to(s["out"].dtype))


def _select(s):
    case = s["case"]
    n, b, v, c = case["groups"], case["beams"], case["vocab"], case["count"]
    # scores that lie near each other decide whole numbers: 64 bits
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    score = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))) + s["scores"].double()[..., None]
    if s["finished"] is not None:
        stay = torch.where(torch.arange(v, device=DEV) == s["stop"], s["scores"].double()[..., None], torch.full((), -math.inf, dtype=torch.float64, device=DEV))
        score = torch.where(s["finished"].bool()[..., None], stay, score)
    value, at = torch.sort(score.view(n, b * v), dim=1, descending=True, stable=True)
    value, at = value[:, :c], at[:, :c]
    parent, token = at // v, at % v
    s["scores_out"].copy_(value.float())
    s["parent_out"].copy_(parent)
    s["token_out"].copy_(token)
    done = token == s["stop"]
    s["finished_out"].copy_(done if s["finished"] is None else done | torch.gather(s["finished"].bool(), 1, parent))


def _reorder(s):
    case = s["case"]
    n, b, page = case["groups"], case["beams"], case["page"]
    parent, table, length = s["parent"].long(), s["table"], s["length"].long()
    beam = torch.arange(b, device=DEV)
    same = parent[:, :, None] == parent[:, None, :]
    earlier = beam[None, :] < beam[:, None]
    further = (same & earlier).any(2)  # not its parent's first child
    bare = ~(parent[:, None, :] == beam[None, :, None]).any(2)  # no child
    # the i-th further child gets the private pages of the i-th beam without children
    rank, order = further.long().cumsum(1) - 1, torch.sort((~bare).long(), dim=1, stable=True)[1]
    owner = torch.where(further, torch.gather(order, 1, rank.clamp_min(0)), parent)
    wide = (n, b, table.shape[-1])
    old = torch.gather(table, 1, parent[..., None].expand(wide))
    private = torch.gather(table, 1, owner[..., None].expand(wide))
    j = torch.arange(table.shape[-1], device=DEV)[None, None]
    s["table_out"].copy_(torch.where(j < (length // page)[:, None, None], old, private))
    # the rows of the last part page
    last, part = (length // page), length % page
    at = last[:, None, None].expand(n, b, 1)
    to, frm = torch.gather(private, 2, at)[..., 0], torch.gather(old, 2, at)[..., 0]
    g, r, t = torch.nonzero(further[:, :, None] & (torch.arange(page, device=DEV)[None, None] < part[:, None, None]), as_tuple=True)
    to, frm = to[g, r].long(), frm[g, r].long()
    s["k"][:, to, :, t] = s["k"][:, frm, :, t]
    s["v"][:, to, :, t] = s["v"][:, frm, :, t]
    state = torch.gather(s["state"], 1, parent[..., None].expand(n, b, case["words"]))
    state.scatter_(2, s["place"].long()[:, None, None].expand(n, b, 1), s["token"][..., None])
    s["state_out"].copy_(state)


# ------------------------------------------------------------------ work
def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "select":
        n = case["groups"] * case["beams"]
        return {"bytes": float(size * n * case["vocab"] + 8 * n + 16 * case["groups"] * case["count"]), "flops": 5.0 * n * case["vocab"]}
    if kind == "reorder":
        b, page = case["beams"], case["page"]
        copies = b * (1.0 - 1.0 / b) ** b  # beams without children, of random parents
        rows = sum(n % page for n in _group_lens(case)) * copies * case["layers"] * case["kv_heads"]
        most = -(-(case["length"] + 1) // page)
        return {"bytes": 2.0 * 2 * rows * case["dim"] * size + 2.0 * 4 * case["groups"] * b * (most + case["words"]), "flops": 0.0}
    new, lens = _lens(case)
    q = case["q_heads"] * case["dim"]
    kv = 2 * case["kv_heads"] * case["dim"]
    if kind == "append":
        turned = sum(new) * case["rot"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2.0 * size * sum(new) * (q + kv) + 4.0 * sum(new), "flops": 3.0 * turned}
    pages = sum(-(-n // case["page"]) for n in lens)
    pairs = sum(k * (n - k) + (k * (k + 1) // 2 if not case["tree"] else k * k) for k, n in zip(new, lens))
    return {"bytes": float(size * (kv * sum(lens) + 2 * q * sum(new)) + 4 * pages), "flops": 4.0 * q * pairs}


# ------------------------------------------------------------------ float64 restatements
F64 = torch.float64


def _turn64(x, position, case):
    y = x.to(F64).clone()
    half = case["rot"] // 2
    for i in range(half):
        a = position.to(F64) * THETA ** (-2.0 * i / case["rot"])
        cos, sin = torch.cos(a)[:, None], torch.sin(a)[:, None]
        p, q = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
        u, w = x[..., p].to(F64), x[..., q].to(F64)
        y[..., p], y[..., q] = u * cos - w * sin, u * sin + w * cos
    return y


def _append64(case, d):
    new, lens = _lens(case)
    place = np.concatenate([np.arange(n - k, n) for k, n in zip(new, lens)])
    seq = np.repeat(np.arange(case["seqs"]), new)
    position = torch.from_numpy(place).to(DEV) if d["position"] is None else d["position"]
    page = torch.from_numpy(d["table"].cpu().numpy()[seq, place // case["page"]]).long().to(DEV)
    slot = torch.from_numpy(place % case["page"]).to(DEV)
    k, v = d["cache_k"].to(F64), d["cache_v"].to(F64)
    k[page, :, slot] = _turn64(d["k"], position, case)
    v[page, :, slot] = d["v"].to(F64)
    return {"q": _turn64(d["q"], position, case), "k": k, "v": v}


def _attention64(case, d):
    new, lens = _lens(case)
    group, page, dim = case["q_heads"] // case["kv_heads"], case["page"], case["dim"]
    out = torch.empty_like(d["q"], dtype=F64)
    at = 0
    for s in range(case["seqs"]):
        n, k = lens[s], new[s]
        pages = d["table"][s, : -(-n // page)].long()
        sees = torch.ones(k, n, dtype=torch.bool, device=DEV)
        if d["mask"] is None:
            sees[:, n - k:] = torch.tril(torch.ones(k, k, dtype=torch.bool, device=DEV))
        else:
            words = d["mask"][at: at + k].cpu().numpy().view(np.uint8)
            sees[:, n - k:] = torch.from_numpy(np.unpackbits(words, axis=1, bitorder="little")[:, :k].astype(bool)).to(DEV)
        for h in range(case["kv_heads"]):
            key = d["cache_k"][pages, h].reshape(-1, dim)[:n].to(F64)
            val = d["cache_v"][pages, h].reshape(-1, dim)[:n].to(F64)
            for g in range(h * group, (h + 1) * group):
                z = (d["q"][at: at + k, g].to(F64) @ key.t().contiguous()) / math.sqrt(dim)
                out[at: at + k, g] = torch.softmax(z.masked_fill(~sees, -math.inf), -1) @ val
        at += k
    return out


def _select64(case, d):
    best = []
    for g in range(case["groups"]):
        lp = torch.log_softmax(d["logits"][g].to(F64), -1) + d["scores"][g].to(F64)[:, None]
        if d["finished"] is not None:
            done = d["finished"][g].bool()
            lp[done] = -math.inf
            lp[done, d["stop"]] = d["scores"][g].to(F64)[done]
        best.append(torch.topk(lp.flatten(), case["count"])[0])
    return {"scores": torch.stack(best), "parent": None, "token": None, "finished": None}


def _reorder64(case, d):
    n, b, page = case["groups"], case["beams"], case["page"]
    parent, lens = d["parent"].cpu().numpy(), _group_lens(case)
    table = d["table"].cpu().numpy().reshape(n, b, -1)
    k, v = d["k"].to(F64), d["v"].to(F64)
    for g in range(n):
        full, part = lens[g] // page, lens[g] % page
        bare = [r for r in range(b) if r not in parent[g]]
        seen = set()
        for r in range(b):
            p = int(parent[g, r])
            if p in seen:
                to, frm = int(table[g, bare.pop(0), full]), int(table[g, p, full])
                k[:, to, :, :part] = d["k"][:, frm, :, :part].to(F64)
                v[:, to, :, :part] = d["v"][:, frm, :, :part].to(F64)
            seen.add(p)
    return {"table": None, "state": None, "k": k, "v": v}


def exact(case, seed):
    d = _inputs(case, seed)
    return {"append": _append64, "attention": _attention64, "select": _select64, "reorder": _reorder64}[case["kind"]](case, d)
