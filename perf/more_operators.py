"""The operators for decoding over long and shared contexts in a paged key/value cache, as a decoding program calls them.

Each case is one call through the Python binding (`mit2cfm.Context`), on buffers that lie on the GPU:

  norm    kv_norm_append_device: each head's new query and key normalised, rotated, keys and values into the pages
  prefix  kv_prefix_attention_device: attention of new rows whose sequences share their first rows, in groups
  weigh   kv_weigh_device: what attention weight the new rows give to each cached row, added up
  evict   kv_evict_device: rows of least accumulated weight leave every layer's cache

Sizes are the GPT decoder's (20 heads of 64, 24 layers), the estimator's (8 heads of 64) or generic ones (32 query
heads on 8 key heads of 128); `draw` spreads over the same ranges.  The plain forms are elementary torch operations;
`exact` restates each operator in float64 from its definition.
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
EPS = 1e-6


# ------------------------------------------------------------------ the cases
def listed():
    gpt = dict(q_heads=20, kv_heads=20, dim=64, dtype="f32", page=64)
    wide = dict(q_heads=32, kv_heads=8, dim=128, dtype="bf16")
    return [
        # one token of three sequences with the GPT decoder's heads: the smallest call
        dict(name="norm_step_3", kind="norm", seqs=3, new=1, length=703, ragged=False, rot=64, interleaved=False, centered=False, per_head=False, **gpt),
        # further pieces of a batch's prompts, part rotation of neighbours, a layer norm with weights of each head
        dict(name="norm_pieces_7", kind="norm", seqs=7, new=129, length=1500, ragged=True, rot=64, interleaved=True, centered=True, per_head=True, page=16,
             q_heads=24, kv_heads=4, dim=96, dtype="f16"),
        # prompts of a batch in one call, lengths as they come
        dict(name="norm_prompts_9", kind="norm", seqs=9, new=2047, length=2900, ragged=True, rot=128, interleaved=False, centered=False, per_head=False, page=32, **wide),
        # hypotheses of a search over one prompt, fp32 as the GPT decoder keeps it
        dict(name="prefix_beams_8", kind="prefix", groups=1, seqs=8, new=1, shared=653, length=801, ragged=False, tree=False, **gpt),
        # a serving batch that answers from one long instruction, lengths as they come
        dict(name="prefix_batch_64", kind="prefix", groups=1, seqs=64, new=1, shared=8191, length=8790, ragged=True, tree=False, page=16, **wide),
        # several instructions, drafted trees checked against each sequence's cache
        dict(name="prefix_trees_4x12", kind="prefix", groups=4, seqs=48, new=9, shared=2903, length=3300, ragged=True, tree=True, page=32, **dict(wide, dtype="f16")),
        # the beams' weights after a step
        dict(name="weigh_step_3", kind="weigh", seqs=3, new=1, length=703, ragged=False, last=0, decay=1.0, **gpt),
        # a serving batch, one token each
        dict(name="weigh_batch_64", kind="weigh", seqs=64, new=1, length=8191, ragged=True, last=0, decay=0.97, page=16, **wide),
        # prompts, all of whose rows count
        dict(name="weigh_prompts_4", kind="weigh", seqs=4, new=1029, length=2047, ragged=True, last=0, decay=1.0, page=32, **dict(wide, dtype="f16")),
        # one row leaves at each step of a full cache, in all layers
        dict(name="evict_step_3", kind="evict", seqs=3, layers=24, length=704, keep=703, first=4, recent=128, ragged=False, born=True, **gpt),
        # prompts cut to a quarter
        dict(name="evict_prompts_8", kind="evict", seqs=8, layers=4, length=8191, keep=2048, first=16, recent=255, ragged=True, born=False, page=16, **wide),
        # one long context cut to half
        dict(name="evict_long_1", kind="evict", seqs=1, layers=3, length=131001, keep=65537, first=64, recent=1024, ragged=False, born=True, page=64, **wide),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["norm", "prefix", "prefix", "weigh", "evict"])
    heads = rng.choice([(20, 20, 64), (8, 8, 64), (32, 8, 128), (24, 4, 96), (16, 2, 128), (7, 1, 32)])
    dtype, page = rng.choice(["f32", "f16", "bf16"]), rng.choice([8, 16, 32, 64, 128])
    form = dict(q_heads=heads[0], kv_heads=heads[1], dim=heads[2], dtype=dtype, page=page)
    ragged = rng.random() < 0.7
    if kind == "norm":
        seqs = log(1, 64)
        new = log(1, max(2, 6000 // seqs))
        return dict(kind=kind, seqs=seqs, new=new, length=new + log(1, 2000), ragged=ragged, rot=2 * rng.randint(0, heads[2] // 2),
                    interleaved=rng.random() < 0.5, centered=rng.random() < 0.3, per_head=rng.random() < 0.3, **form)
    if kind == "prefix":
        groups, tree = log(1, 8), rng.random() < 0.4
        seqs = groups * log(1, max(1, 64 // groups))
        new = rng.randint(2, 17) if tree else rng.choice([1, 1, 1, log(2, 40)])
        shared = log(30, min(20000, 60000 // groups))
        return dict(kind=kind, groups=groups, seqs=seqs, new=new, shared=shared, length=shared + new + log(1, max(2, min(1200, 40000 // seqs))), ragged=ragged,
                    tree=tree, **form)
    if kind == "weigh":
        if rng.random() < 0.6:
            seqs = log(1, 64)
            return dict(kind=kind, seqs=seqs, new=1, length=log(1, min(100000, 180000 // seqs)), ragged=ragged, last=0, decay=rng.choice([1.0, 0.9]), **form)
        seqs = log(1, 7)
        new = log(2, 700)
        return dict(kind=kind, seqs=seqs, new=new, length=new + log(1, 2000), ragged=ragged, last=rng.choice([0, 0, 32]), decay=rng.choice([1.0, 0.9]), **form)
    seqs = log(1, 16)
    length = log(20, min(60000, 120000 // seqs))
    row = heads[1] * heads[2] * (4 if dtype == "f32" else 2) * 2
    layers = max(1, min(rng.randint(1, 24), int(1.5e9 / (row * seqs * length))))
    keep = max(1, int(length * rng.choice([0.25, 0.5, 0.9])) if rng.random() < 0.7 else length - log(1, min(64, length - 1)))
    return dict(kind=kind, seqs=seqs, layers=layers, length=length, keep=keep, first=rng.randint(0, 1 + keep // 8), recent=rng.randint(0, 1 + keep // 4),
                ragged=ragged, born=rng.random() < 0.5, **form)


# ------------------------------------------------------------------ inputs
def _lens(case):
    """(new rows, cached rows with them) of each sequence; a ragged batch's first is the largest."""
    n = case["seqs"]
    u = [((5 * s) % n) / n if case["ragged"] else 0.0 for s in range(n)]
    if case["kind"] == "evict":
        return [0] * n, [max(1, round(case["length"] * (1.0 - 0.6 * x))) for x in u]
    new = [1 + int((case["new"] - 1) * (1.0 - 0.6 * x)) for x in u]
    if case["kind"] == "prefix":  # rows of their own: those after the shared ones
        return new, [case["shared"] + max(k, round((case["length"] - case["shared"]) * (1.0 - 0.9 * x))) for k, x in zip(new, u)]
    return new, [max(k, round(case["length"] * (1.0 - 0.6 * x))) for k, x in zip(new, u)]


def _keeps(case):
    """Rows that stay of each sequence, in the proportion of its length."""
    return [max(1, n * case["keep"] // case["length"]) for n in _lens(case)[1]]


def _trees(seqs, new, rng):
    """Random trees over each sequence's new rows: whether row i's path from the root holds row j."""
    n = max(new)
    sees = np.zeros((seqs, n, n), bool)
    every = np.arange(seqs)
    for i in range(n):
        parent = rng.integers(max(-1, i - 6), i, seqs) if i else np.full(seqs, -1)
        has = parent >= 0
        sees[has, i] = sees[every[has], parent[has]]
        sees[:, i, i] = True
    return sees


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _tables(case, lens, rng):
    """Page tables [seqs][entries] over random pages; of a group's shared rows the full pages are the same."""
    page, seqs = case["page"], case["seqs"]
    most = -(-max(lens) // page)
    table = np.zeros((seqs, most), np.int64)
    each = seqs // case["groups"] if case["kind"] == "prefix" else 1
    full = case["shared"] // page if case["kind"] == "prefix" else 0
    held = [-(-n // page) for n in lens]
    pages = sum(held) - (seqs - seqs // each) * full
    ids = rng.permutation(pages)
    at = 0
    for s in range(seqs):
        if s % each == 0:
            table[s, :full] = ids[at: at + full]
            at += full
        else:
            table[s, :full] = table[s - s % each, :full]
        table[s, full: held[s]] = ids[at: at + held[s] - full]
        at += held[s] - full
    return table, pages


def _inputs(case, seed):
    """Inputs from the seed alone."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, dtype, page, seqs = case["kind"], TYPES[case["dtype"]], case["page"], case["seqs"]
    qh, kvh, dim = case["q_heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    new, lens = _lens(case)
    table, pages = _tables(case, lens, rng)
    d = dict(table=_ints(table), length=_ints(lens))
    if kind == "evict":
        shape = (case["layers"], pages, kvh, page, dim)
        d.update(k=normal(*shape), v=normal(*shape), keep=_ints(_keeps(case)), born=None, now=None)
        wide = (case["layers"], seqs, kvh, table.shape[1] * page)
        # weights as they add up: a few rows have most of it
        d["weights"] = torch.exp(2.0 * torch.randn(*wide, generator=g, device=DEV))
        if case["born"]:
            # earlier evictions have left gaps in the positions, and rows out of their order
            n = int(1.5 * case["length"]) + 16
            ages = np.stack([np.sort(rng.permutation(n)[: wide[3]]) if n >= wide[3] else np.arange(wide[3]) for _ in range(min(8, seqs * kvh))])
            ages = np.concatenate([rng.permuted(ages[:, : wide[3] // 2], axis=1), ages[:, wide[3] // 2:]], 1)
            at = np.arange(case["layers"] * seqs * kvh) % len(ages)
            d["born"] = _ints(ages[at].reshape(wide))
            d["now"] = d["born"].amax(dim=(0, 2, 3)).add_(1).int() if seqs > 1 else d["born"].amax().reshape(1).add_(1).int()
        return d
    start, rows = np.cumsum([0] + new), sum(new)
    d.update(start=_ints(start), q=normal(rows, qh, dim), mask=None, position=None, cache_k=normal(pages, kvh, page, dim))
    if kind == "norm":
        heads = (qh, kvh) if case["per_head"] else (1, 1)
        d.update(cache_v=normal(pages, kvh, page, dim), k=normal(rows, kvh, dim) * 3.0, v=normal(rows, kvh, dim),
                 q_weight=1.0 + 0.2 * normal(heads[0], dim), k_weight=1.0 + 0.2 * normal(heads[1], dim))
        return d
    if kind == "prefix":
        d["cache_v"] = normal(pages, kvh, page, dim)
        if case["shared"] % page:  # the last shared rows lie in each sequence's own page
            each, full, part = seqs // case["groups"], case["shared"] // page, case["shared"] % page
            for s in range(seqs):
                if s % each:
                    for x in (d["cache_k"], d["cache_v"]):
                        x[int(table[s, full]), :, :part] = x[int(table[s - s % each, full]), :, :part]
        d["group"] = _ints(np.arange(case["groups"] + 1) * (seqs // case["groups"]))
        d["shared"] = _ints([case["shared"]] * case["groups"])
        if case["tree"]:
            sees = _trees(seqs, new, rng)
            bits = np.zeros((rows, -(-max(new) // 32) * 32), bool)
            for s in range(seqs):
                bits[start[s]: start[s + 1], : new[s]] = sees[s, : new[s], : new[s]]
            d["mask"] = _ints(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
        return d
    # weigh: queries whose attention is not even, the log sums that the attention leaves, what had added up before
    d["q"] = d["q"] * 2.0
    d["weights"] = torch.rand(seqs, kvh, table.shape[1] * page, generator=g, device=DEV) * 4.0
    d["lse"] = torch.empty(rows, qh, device=DEV)
    for s in range(seqs):
        n, k = lens[s], new[s]
        key = d["cache_k"][d["table"][s, : -(-n // page)].long()].transpose(0, 1).reshape(kvh, -1, dim)[:, :n].float()
        q = d["q"][start[s]: start[s + 1]].float().view(k, kvh, qh // kvh, dim).permute(1, 2, 0, 3).reshape(kvh, -1, dim)
        z = torch.matmul(q, key.transpose(1, 2).contiguous()).view(kvh, qh // kvh, k, n) / math.sqrt(dim)
        late = torch.arange(n, device=DEV)[None] > torch.arange(n - k, n, device=DEV)[:, None]
        d["lse"][start[s]: start[s + 1]] = torch.logsumexp(z.masked_fill_(late, -math.inf), -1).permute(2, 0, 1).reshape(k, qh)
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
    qh, kvh, d = case["q_heads"], case["kv_heads"], case["dim"]

    def at(name):
        return s[name].data_ptr() if s.get(name) is not None else None

    def workspace(a, n):
        s["workspace"] = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
        a.workspace, a.workspace_bytes = at("workspace"), s["workspace"].numel()

    keys, values = ("k", "v") if kind == "evict" else ("cache_k", "cache_v")
    cache = mit2cfm.KvCache(k=at(keys), v=at(values) or at(keys), table=at("table"), pages=s[keys].shape[-4], page_rows=case["page"], kv_heads=kvh,
                            head_dim=d, table_stride=s["table"].shape[1], dtype=mit2cfm.DTYPES[case["dtype"]])
    new, lens = _lens(case)
    if kind == "evict":
        a = mit2cfm.KvEvict(seqs=case["seqs"], layers=case["layers"], layer_stride=s["k"].stride(0), length=at("length"), keep=at("keep"),
                            first_rows=case["first"], last_rows=case["recent"], max_length=max(lens), weights=at("weights"),
                            weights_out=at("weights_out"), weight_stride=s["weights"].shape[-1], born=at("born"), born_out=at("born_out"), now=at("now"),
                            length_out=at("length_out"))
        workspace(a, mit2cfm.kv_evict_workspace(cache, a))
        return dict(cache=cache, args=a)
    rows = mit2cfm.KvRows(start=at("start"), length=at("length"), seqs=case["seqs"], rows=sum(new), max_length=max(lens))
    if kind == "norm":
        a = mit2cfm.KvAppend(k=at("k"), v=at("v"), k_row=kvh * d, k_head=d, v_row=kvh * d, v_head=d, q=at("q"), q_out=at("out"), q_row=qh * d,
                             q_head=d, q_out_row=qh * d, q_out_head=d, q_heads=qh, position=at("position"), rotary_dim=case["rot"],
                             interleaved=int(case["interleaved"]), theta=THETA)
        n = mit2cfm.KvNorm(q_weight=at("q_weight"), k_weight=at("k_weight"), q_weight_head=d if case["per_head"] else 0,
                           k_weight_head=d if case["per_head"] else 0, weight_dtype=mit2cfm.DTYPES[case["dtype"]], centered=int(case["centered"]), eps=EPS)
        return dict(cache=cache, rows=rows, args=a, more=n)
    if kind == "weigh":
        a = mit2cfm.KvWeigh(q=at("q"), q_row=qh * d, q_head=d, q_heads=qh, scale=1.0 / math.sqrt(d), last_rows=case["last"], lse=at("lse"),
                            weights=at("weights"), weights_out=at("weights_out"), weight_stride=s["weights"].shape[-1], decay=case["decay"])
        return dict(cache=cache, rows=rows, args=a)
    a = mit2cfm.KvAttention(q=at("q"), out=at("out"), q_row=qh * d, q_head=d, out_row=qh * d, out_head=d, q_heads=qh, scale=1.0 / math.sqrt(d),
                            mask=at("mask"), mask_words=0 if s["mask"] is None else s["mask"].shape[1])
    p = mit2cfm.KvPrefix(group=at("group"), shared=at("shared"), groups=case["groups"], max_shared=case["shared"], lse=at("lse"))
    workspace(a, mit2cfm.kv_prefix_attention_workspace(cache, rows, qh, p))
    return dict(cache=cache, rows=rows, args=a, more=p)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind == "evict":
        s["length_out"] = torch.empty_like(s["length"])
        # (places past the rows that stay are not written)
        s["weights_out"] = s["weights"].clone()
        s["born_out"] = None if s["born"] is None else s["born"].clone()
    elif kind == "weigh":
        s["weights_out"] = s["weights"].clone()
    else:
        s["out"] = torch.empty_like(s["q"])
        if kind == "prefix":
            s["lse"] = torch.empty(s["q"].shape[:2], device=DEV)
    if own:
        s["plan"] = _plan(s)
    torch.cuda.synchronize()  # a context works on a stream of its own
    return s


# ------------------------------------------------------------------ one pass
def _outputs(s):
    kind = s["case"]["kind"]
    if kind == "norm":
        return {"q": s["out"], "k": s["cache_k"], "v": s["cache_v"]}
    if kind == "prefix":
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "weigh":
        return {"weights": s["weights_out"]}
    r = {"length": s["length_out"], "weights": s["weights_out"], "k": s["k"], "v": s["v"]}
    return r if s["born"] is None else dict(r, born=s["born_out"])


def run(s):
    kind = s["case"]["kind"]
    if own:
        p = s["plan"]
        if kind == "norm":
            s["ctx"].kv_norm_append_device(p["cache"], p["rows"], p["args"], p["more"])
        elif kind == "prefix":
            s["ctx"].kv_prefix_attention_device(p["cache"], p["rows"], p["args"], p["more"])
        elif kind == "weigh":
            s["ctx"].kv_weigh_device(p["cache"], p["rows"], p["args"])
        else:
            s["ctx"].kv_evict_device(p["cache"], p["args"])
        return _outputs(s)
    {"norm": _norm, "prefix": _prefix, "weigh": _weigh, "evict": _evict}[kind](s)
    return _outputs(s)


# ------------------------------------------------------------------ plain forms
def _places(s):
    """Each new row's sequence and its place there."""
    start, length = s["start"].long(), s["length"].long()
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(start[1:], row, right=True)
    return seq, row - start[seq], length[seq] - (start[seq + 1] - start[seq])


def _normed(x, weight, case):
    """[rows][heads][dim] in 32 bits, normalised over dim."""
    y = x.float()
    if case["centered"]:
        y = y - y.mean(-1, keepdim=True)
    return y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(y, position, case):
    half = case["rot"] // 2
    if half == 0:
        return y
    # far positions: the angle in 64 bits
    a = position.double()[:, None] * torch.exp(torch.arange(half, device=DEV).double() * (-2.0 * math.log(THETA) / case["rot"]))
    cos, sin = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    r, rest = y[..., : case["rot"]], y[..., case["rot"]:]
    if case["interleaved"]:
        u, w = r[..., 0::2], r[..., 1::2]
        r = torch.stack([u * cos - w * sin, w * cos + u * sin], -1).flatten(-2)
    else:
        u, w = r[..., :half], r[..., half:]
        r = torch.cat([u * cos - w * sin, w * cos + u * sin], -1)
    return torch.cat([r, rest], -1)


def _norm(s):
    case = s["case"]
    seq, i, before = _places(s)
    place = before + i
    position = place if s["position"] is None else s["position"]
    page = s["table"].long()[seq, place // case["page"]]
    s["cache_k"][page, :, place % case["page"]] = _rotated(_normed(s["k"], s["k_weight"], case), position, case).to(s["k"].dtype)
    s["cache_v"][page, :, place % case["page"]] = s["v"]
    s["out"].copy_(_rotated(_normed(s["q"], s["q_weight"], case), position, case).to(s["out"].dtype))


def _scores(s, cache):
    """Every sequence's scores in 32 bits [seqs][kv heads][group * new][cached rows], and where its rows lie: -inf for what is not seen."""
    case = s["case"]
    seqs, kvh, d = case["seqs"], case["kv_heads"], case["dim"]
    group, new = case["q_heads"] // kvh, case["new"]
    seq, i, _ = _places(s)
    start = s["start"].long()
    k = cache[s["table"].long()].transpose(1, 2).reshape(seqs, kvh, -1, d).float()
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
    return score.masked_fill(~sees, -math.inf), seq, i


def _prefix(s):
    case = s["case"]
    seqs, kvh, d = case["seqs"], case["kv_heads"], case["dim"]
    group, new = case["q_heads"] // kvh, case["new"]
    score, seq, i = _scores(s, s["cache_k"])
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = s["cache_v"][s["table"].long()].transpose(1, 2).reshape(seqs, kvh, -1, d).float()
    out = torch.matmul(p, v) / total.clamp_min(1e-30)
    lse = (top + torch.log(total))[..., 0].view(seqs, kvh, group, new).permute(0, 3, 1, 2).reshape(seqs, new, case["q_heads"])
    out = out.view(seqs, kvh, group, new, d).permute(0, 3, 1, 2, 4).reshape(seqs, new, case["q_heads"], d)
    s["out"].copy_(out[seq, i].to(s["out"].dtype))
    s["lse"].copy_(lse[seq, i])


def _weigh(s):
    case = s["case"]
    seqs, kvh = case["seqs"], case["kv_heads"]
    group, new = case["q_heads"] // kvh, case["new"]
    score, seq, i = _scores(s, s["cache_k"])
    n = score.shape[-1]
    lse = torch.full((seqs, new, case["q_heads"]), math.inf, device=DEV)
    lse[seq, i] = s["lse"]
    count = (s["start"][1:] - s["start"][:-1]).long()
    if case["last"]:
        early = torch.arange(new, device=DEV)[None] < count[:, None] - case["last"]
        lse = lse.masked_fill(early[..., None], math.inf)
    lse = lse.view(seqs, new, kvh, group).permute(0, 2, 3, 1).reshape(seqs, kvh, group * new, 1)
    got = torch.exp(score - lse).sum(2)
    length = s["length"].long()[:, None, None]
    place = torch.arange(n, device=DEV)[None, None]
    before = torch.where(place < length - count[:, None, None], s["weights"][..., :n] * case["decay"], torch.zeros((), device=DEV))
    s["weights_out"][..., :n] = torch.where(place < length, before + got, s["weights_out"][..., :n])


def _evict(s):
    case = s["case"]
    layers, seqs, kvh, page = case["layers"], case["seqs"], case["kv_heads"], case["page"]
    n = s["weights"].shape[-1]
    length, keep = s["length"].long()[:, None], s["keep"].long()[:, None]
    place = torch.arange(n, device=DEV)[None]
    stay = (place < case["first"])[None, :, None].expand(layers, seqs, kvh, n)
    if s["born"] is None:
        stay = stay | (place >= length - case["recent"])[None, :, None]
    else:
        stay = stay | (s["born"].long() >= s["now"].long()[None, :, None, None] - case["recent"])
    # values next to the border decide whole numbers: 64 bits
    key = s["weights"].double().masked_fill(stay, math.inf).masked_fill((place >= length)[None, :, None], -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    most = torch.minimum(length, keep)
    inside = (place < most)[None, :, None].expand(layers, seqs, kvh, n)
    kept = torch.zeros(layers, seqs, kvh, n, dtype=torch.bool, device=DEV).scatter_(-1, order, inside)
    # the places that get free below `keep`, and the rows that stay from there on: the i-th goes to the i-th
    to = torch.nonzero(inside & ~kept)
    frm = torch.nonzero(kept & ~inside)
    layer, seq, head, dst = to.unbind(1)
    src = frm[:, 3]
    table = s["table"].long()
    for x in (s["k"], s["v"]):
        x[layer, table[seq, dst // page], head, dst % page] = x[layer, table[seq, src // page], head, src % page]
    s["length_out"].copy_(most[:, 0])
    for name in ("weights", "born"):
        if s[name] is not None:
            moved = s[name].clone()
            moved[layer, seq, head, dst] = s[name][layer, seq, head, src]
            s[name + "_out"].copy_(torch.where(inside, moved, s[name + "_out"]))


# ------------------------------------------------------------------ work
def _moves(case):
    """Rows that move of a head in one layer, weights and ages at random: of those that stay, the ones from `keep` on."""
    total = 0.0
    for n, m in zip(_lens(case)[1], _keeps(case)):
        m = min(n, m)
        first, recent = min(case["first"], m), min(case["recent"], max(m - case["first"], 0))
        middle = max(n - first - recent, 1)
        total += min(recent, n - m) + max(n - m - recent, 0) * (m - first - recent) / middle
    return total


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    new, lens = _lens(case)
    q = case["q_heads"] * case["dim"]
    kv = 2 * case["kv_heads"] * case["dim"]
    if kind == "norm":
        return {"bytes": 2.0 * size * sum(new) * (q + kv) + 4.0 * sum(new), "flops": sum(new) * (q + kv / 2) * 7.0}
    if kind == "evict":
        heads = case["layers"] * case["kv_heads"]
        side = 8.0 if case["born"] else 4.0
        return {"bytes": heads * (2.0 * 2 * size * case["dim"] * _moves(case) + side * sum(lens) + side * sum(min(a, b) for a, b in zip(lens, _keeps(case)))),
                "flops": 0.0}
    pages = sum(-(-n // case["page"]) for n in lens)
    if kind == "prefix":
        cached = case["groups"] * case["shared"] + sum(n - case["shared"] for n in lens)
        pairs = sum(k * (n - k) + (k * (k + 1) // 2 if not case["tree"] else k * k) for k, n in zip(new, lens))
        return {"bytes": float(size * (kv * cached + 2 * q * sum(new)) + 4 * pages + 4 * sum(new) * case["q_heads"]), "flops": 4.0 * q * pairs}
    used = [min(k, case["last"] or k) for k in new]
    pairs = sum(u * (n - u) + u * (u + 1) // 2 for u, n in zip(used, lens))
    return {"bytes": float(size * (kv // 2 * sum(lens) + q * sum(used)) + 4 * pages + 4 * sum(used) * case["q_heads"] + 8 * sum(lens) * case["kv_heads"]),
            "flops": 2.0 * q * pairs}


# ------------------------------------------------------------------ float64 restatements
F64 = torch.float64


def _heads64(x, weight, position, case):
    """The definition, a pair of elements at a time."""
    y = x.to(F64)
    if case["centered"]:
        y = y - y.sum(-1, keepdim=True) / case["dim"]
    y = y * torch.rsqrt((y ** 2).sum(-1, keepdim=True) / case["dim"] + EPS) * weight.to(F64)
    out = y.clone()
    half = case["rot"] // 2
    for i in range(half):
        a = position.to(F64) * THETA ** (-2.0 * i / case["rot"])
        cos, sin = torch.cos(a)[:, None], torch.sin(a)[:, None]
        p, r = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
        out[..., p], out[..., r] = y[..., p] * cos - y[..., r] * sin, y[..., p] * sin + y[..., r] * cos
    return out


def _norm64(case, d):
    new, lens = _lens(case)
    place = np.concatenate([np.arange(n - k, n) for k, n in zip(new, lens)])
    seq = np.repeat(np.arange(case["seqs"]), new)
    position = torch.from_numpy(place).to(DEV)
    page = torch.from_numpy(d["table"].cpu().numpy()[seq, place // case["page"]]).long().to(DEV)
    slot = torch.from_numpy(place % case["page"]).to(DEV)
    k, v = d["cache_k"].to(F64), d["cache_v"].to(F64)
    k[page, :, slot] = _heads64(d["k"], d["k_weight"], position, case)
    v[page, :, slot] = d["v"].to(F64)
    return {"q": _heads64(d["q"], d["q_weight"], position, case), "k": k, "v": v}


def _each64(case, d):
    """(sequence, its first new row, new rows, length, key head, query head, scores [new][length] with -inf, pages)."""
    new, lens = _lens(case)
    group, page, dim = case["q_heads"] // case["kv_heads"], case["page"], case["dim"]
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
            for g in range(h * group, (h + 1) * group):
                z = (d["q"][at: at + k, g].to(F64) @ key.t().contiguous()) / math.sqrt(dim)
                yield s, at, k, n, h, g, z.masked_fill(~sees, -math.inf), pages
        at += k


def _prefix64(case, d):
    out, lse = torch.empty_like(d["q"], dtype=F64), torch.empty(d["q"].shape[:2], dtype=F64, device=DEV)
    for s, at, k, n, h, g, z, pages in _each64(case, d):
        val = d["cache_v"][pages, h].reshape(-1, case["dim"])[:n].to(F64)
        out[at: at + k, g] = torch.softmax(z, -1) @ val
        lse[at: at + k, g] = torch.logsumexp(z, -1)
    return {"out": out, "lse": lse}


def _weigh64(case, d):
    new, lens = _lens(case)
    w = d["weights"].to(F64)
    for s in range(case["seqs"]):
        w[s, :, : lens[s] - new[s]] *= case["decay"]
        w[s, :, lens[s] - new[s]: lens[s]] = 0.0
    for s, at, k, n, h, g, z, _ in _each64(case, d):
        u = min(k, case["last"] or k)
        w[s, h, :n] += torch.exp(z[k - u:] - d["lse"][at + k - u: at + k, g].to(F64)[:, None]).sum(0)
    return {"weights": w}


def _evict64(case, d):
    lens, keeps, page = _lens(case)[1], _keeps(case), case["page"]
    table, weights = d["table"].cpu().numpy(), d["weights"].cpu().numpy().astype(np.float64)
    born = None if d["born"] is None else d["born"].cpu().numpy().astype(np.int64)
    now = None if born is None else d["now"].cpu().numpy().astype(np.int64)
    k, v, w = d["k"].to(F64), d["v"].to(F64), weights.copy()
    frm, to = [], []
    for layer in range(case["layers"]):
        for s, (n, m) in enumerate(zip(lens, keeps)):
            m = min(n, m)
            for h in range(case["kv_heads"]):
                key = weights[layer, s, h, :n].copy()
                key[: case["first"]] = np.inf
                if born is None:
                    key[max(0, n - case["recent"]):] = np.inf
                else:
                    key[born[layer, s, h, :n] >= now[s] - case["recent"]] = np.inf
                stays = np.zeros(n, bool)
                stays[np.lexsort((np.arange(n), -key))[:m]] = True
                dst, src = np.flatnonzero(~stays[:m]), m + np.flatnonzero(stays[m:])
                w[layer, s, h, dst] = weights[layer, s, h, src]
                line = np.full(len(dst), layer), np.full(len(dst), h)
                to.append(np.stack([line[0], table[s, dst // page], line[1], dst % page]))
                frm.append(np.stack([line[0], table[s, src // page], line[1], src % page]))
    to, frm = (tuple(torch.from_numpy(np.concatenate(x, 1)).long().to(DEV)) for x in (to, frm))
    k[to], v[to] = d["k"][frm].to(F64), d["v"][frm].to(F64)
    r = {"length": None, "weights": torch.from_numpy(w).to(DEV), "k": k, "v": v}
    return r if born is None else dict(r, born=None)


def exact(case, seed):
    d = _inputs(case, seed)
    return {"norm": _norm64, "prefix": _prefix64, "weigh": _weigh64, "evict": _evict64}[case["kind"]](case, d)
