"""The operators of batched decoding over a paged KV cache: what is measured,
and their plain forms.

  append   per-head RMSNorm of q and k, rotary embedding, the K and V rows
           into the pages (a decode step, or the rows of whole prompts)
  attend   attention of one new token per sequence over its pages, with or
           without the attention weights accumulated per cached row
  evict    the cached rows of least accumulated weight leave the cache
  sample   temperature, top-k, top-p and min-p, and a draw from given
           uniform numbers

Pools are [n_pages][n_kv_heads][page_size][head_dim]; row r of sequence b is
in page table[b][r // page_size].  The plain forms below are elementary torch
operations in 32 bits; with `own` the framework's calls run instead.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_VOCAB = 151936          # the vocabulary of the benchmark's decode step
_EPS = 1e-6
_BASE = 1_000_000.0      # rotary base of the same configuration
_UNIT = 40               # a weight of 1 is 2^40 in the sampler's sums


# ------------------------------------------------------------------- cases
def _attend(name, batch, heads, kv_heads, dim, page, dtype, longest, lens, window=0, accumulate=False):
    return {"name": name, "op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "type": dtype, "longest": longest, "lens": lens, "window": window,
            "accumulate": accumulate}


def _append(name, seqs, tokens, heads, kv_heads, dim, page, dtype, longest, norms=True):
    return {"name": name, "op": "append", "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "type": dtype, "longest": longest, "norms": norms}


def _evict(name, batch, kv_heads, dim, page, dtype, longest, lens, budget, recent, sinks):
    return {"name": name, "op": "evict", "batch": batch, "kv_heads": kv_heads, "dim": dim, "page": page,
            "type": dtype, "longest": longest, "lens": lens, "budget": budget, "recent": recent, "sinks": sinks}


def _sample(name, batch, vocab, settings, spread):
    return {"name": name, "op": "sample", "batch": batch, "vocab": vocab, "settings": settings, "spread": spread}


def listed():
    return [
        # the first tokens of one conversation: nothing but latency
        _attend("attend one short f16", 1, 32, 4, 128, 16, "f16", 37, "even"),
        # an ordinary server: requests of every age, one slot of the batch empty
        _attend("attend batch ragged bf16", 32, 32, 4, 128, 64, "bf16", 4096, "ragged"),
        # one conversation over a whole book: the length itself has to be split
        _attend("attend one long f16", 1, 32, 4, 128, 64, "f16", 131071, "even"),
        # a full server at 16 query heads per kv head (64 query heads of the 94-layer shape)
        _attend("attend full server bf16", 64, 64, 4, 128, 64, "bf16", 8192, "ragged"),
        # the cache in the activations' own type, as the single-sequence path keeps it; only a window is seen
        _attend("attend window f32", 8, 32, 4, 128, 32, "f32", 4099, "ragged", window=2048),
        # the step before an eviction: the weights are accumulated as the rows are read
        _attend("attend accumulate f16", 16, 32, 4, 128, 64, "f16", 4200, "ragged", accumulate=True),
        # one decode step of a full batch, one layer
        _append("append step f16", 64, 64, 32, 4, 128, 64, "f16", 8192),
        # prompts of several requests written in one go
        _append("append prompts bf16", 6, 8191, 32, 4, 128, 64, "bf16", 4000),
        # a long prompt cut to its heavy hitters before decoding starts
        _evict("evict prompt f16", 1, 4, 128, 64, "f16", 32768, "even", 4096, 512, 4),
        # steady state of a bounded cache: every so many steps a few rows leave
        _evict("evict step bf16", 32, 4, 128, 64, "bf16", 2176, "even", 2048, 256, 4),
        # one conversation, the usual settings
        _sample("sample one", 1, _VOCAB, "usual", 3.0),
        # a full batch, every request with its own settings, some unfiltered
        _sample("sample batch mixed", 64, _VOCAB, "mixed", 3.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "evict", "sample", "sample"])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 4, 8])
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    if op == "attend":
        batch = _log(rng, 1, 64)
        gqa = rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
        # the pool holds at most what the full server's does
        most = 64 * 8192 * 4 * 128 // (batch * kv_heads * dim) // (2 if dtype == "f32" else 1)
        longest = _log(rng, 1, max(2, min(131072, most)))
        c = _attend("", batch, gqa * kv_heads, kv_heads, dim, page, dtype, longest, rng.choice(["even", "ragged"]),
                    rng.choice([0, 0, 0, max(1, longest // 3)]), rng.random() < 0.25)
    elif op == "append":
        seqs = _log(rng, 1, 64)
        tokens = seqs if rng.random() < 0.5 else _log(rng, seqs, 8192)
        gqa = rng.choice([1, 2, 4, 5, 8])
        c = _append("", seqs, tokens, gqa * kv_heads, kv_heads, min(dim, 128), page, dtype,
                    -(-tokens // seqs) + _log(rng, 1, 2000), rng.random() < 0.7)
    elif op == "evict":
        batch = _log(rng, 1, 32)
        longest = _log(rng, 64, min(32768, 32 * 4096 * 4 * 128 // (batch * kv_heads * dim)))
        budget = max(8, int(longest * rng.uniform(0.1, 0.97)))
        c = _evict("", batch, kv_heads, dim, page, dtype, longest, rng.choice(["even", "ragged"]), budget,
                   int(budget * rng.uniform(0, 0.5)), rng.choice([0, 1, 4]))
    else:
        c = _sample("", _log(rng, 1, 64), _log(rng, 1000, 200000), rng.choice(["usual", "mixed", "greedy", "free"]),
                    rng.choice([1.0, 2.0, 3.0]))
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _lens(case):
    """Rows of each sequence, from the case alone (prepare() shuffles them): all as long as the longest, or even
    steps up to it, the first slot empty where there are four or more."""
    b, longest = case["batch"], case["longest"]
    if case["lens"] == "even":
        return [longest] * b
    got = [max(1, longest * (i + 1) // b) for i in range(b)]
    if b >= 4:
        got[0] = 0
    return got


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _pool(g, case, batch, rows):
    """K and V pools with a tenth more pages than the sequences need, and a table that hands them out in no order.
    Pages that no sequence has, and what a page holds past its sequence's end, keep the values of earlier ones."""
    width = -(-rows // case["page"])
    n_pages = batch * width + batch * width // 10 + 1
    table = torch.randperm(n_pages, generator=g, device="cuda")[:batch * width].reshape(batch, width)
    shape = (n_pages, case["kv_heads"], case["page"], case["dim"])
    dtype = _TYPES[case["type"]]
    pools = []
    for _ in range(2):
        pool = torch.empty(shape, dtype=dtype, device="cuda")
        for at in range(0, n_pages, 4096):      # in parts: no second pool in 32 bits
            part = pool[at:at + 4096]
            part.copy_(_normal(g, *part.shape))
        pools.append(pool)
    return pools[0], pools[1], table.to(torch.int32).contiguous()


def _address(table, page, rows):
    """Page and place in the page of `rows` [rows] of every sequence."""
    return table.long()[:, rows // page], rows % page


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": dict(case)}
    op = case["op"]
    if op == "sample":
        _prepare_sample(s, case, g)
        return s
    batch = case["seqs"] if op == "append" else case["batch"]
    k, v, table = _pool(g, case, batch, case["longest"])
    s.update(k=k, v=v, table=table)
    shuffled = torch.randperm(batch, generator=g, device="cuda")
    if op == "append":
        _prepare_append(s, case, g)
    else:
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[shuffled].contiguous()
    if op == "attend":
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        # heads of every sharpness: scores of spread 1/2 to 4
        sharp = torch.exp(torch.rand(heads, generator=g, device="cuda") * math.log(8.0)) / 2
        s["q"] = (_normal(g, batch, heads, dim) * sharp[:, None]).contiguous()
        # what lies past a sequence's end was never written, or anything else wrote it
        rows = torch.arange(table.shape[1] * case["page"], device="cuda")
        pg, at = _address(table, case["page"], rows)
        b, r = torch.nonzero(rows[None] >= s["lens"][:, None], as_tuple=True)
        k[pg[b, r], :, at[r]] = float("nan")
        v[pg[b, r], :, at[r]] = float("inf")
        if case["accumulate"]:
            s["acc"] = torch.rand(batch, kv, rows.numel(), generator=g, device="cuda") * case["heads"] / kv
            s["acc_out"] = torch.zeros_like(s["acc"])
    elif op == "evict":
        kv, stride = case["kv_heads"], table.shape[1] * case["page"]
        # accumulated weights fall like a power of their rank; equal ones occur
        w = torch.rand(batch, kv, stride, generator=g, device="cuda") ** -0.7 - 1
        s["acc"] = (torch.floor(w * 4096) / 4096).contiguous()
        # rows of one sequence are of distinct, mostly rising positions (earlier evictions left gaps and moved some)
        p = torch.arange(stride, device="cuda") * 3 + torch.randint(0, 3, (batch, kv, stride), generator=g,
                                                                   device="cuda")
        flip = torch.rand(batch, kv, stride // 2, generator=g, device="cuda") < 0.1
        a, b = p[..., 0:2 * (stride // 2):2].clone(), p[..., 1:2 * (stride // 2):2].clone()
        p[..., 0:2 * (stride // 2):2] = torch.where(flip, b, a)
        p[..., 1:2 * (stride // 2):2] = torch.where(flip, a, b)
        s["pos"] = p.to(torch.int32).contiguous()
        s["next_pos"] = (s["lens"] * 3).to(torch.int32).contiguous()
        s["acc_out"] = torch.zeros_like(s["acc"])
        s["pos_out"] = torch.zeros_like(s["pos"])
        s["lens_out"] = torch.zeros_like(s["lens"])
    if own:
        # the cache object that a server keeps for as long as it runs
        from styx_b200 import ops
        s["kv"] = ops.PagedKV(k, v, table, s["lens"])
    return s


def _prepare_append(s, case, g):
    n, seqs, heads, kv, dim = case["tokens"], case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    # q, k and v lie side by side, as one projection leaves them
    qkv = _normal(g, n, (heads + 2 * kv) * dim)
    s["q"], s["key"], s["value"] = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv * dim, kv * dim], 1))
    s["q_norm"] = torch.rand(dim, generator=g, device="cuda") + 0.5 if case["norms"] else None
    s["k_norm"] = torch.rand(dim, generator=g, device="cuda") + 0.5 if case["norms"] else None
    t = torch.arange(n, device="cuda")
    seq = t * seqs // n                                    # consecutive tokens of a prompt, prompt after prompt
    first = torch.searchsorted(seq, torch.arange(seqs, device="cuda"))
    count = torch.bincount(seq, minlength=seqs)
    before = torch.floor(torch.rand(seqs, generator=g, device="cuda") * (case["longest"] - count + 1)).long()
    s["seq"] = seq.to(torch.int32).contiguous()
    s["row"] = (before[seq] + t - first[seq]).to(torch.int32).contiguous()
    s["lens"] = (before + count).to(torch.int32).contiguous()
    # positions run ahead of rows where rows were evicted
    s["pos"] = (s["row"].long() + (torch.rand(seqs, generator=g, device="cuda") * 100000).long()[seq]).to(
        torch.int32).contiguous()
    s["q_out"] = torch.zeros(n, heads, dim, device="cuda")


def _prepare_sample(s, case, g):
    b, v = case["batch"], case["vocab"]
    x = _normal(g, b, v) * case["spread"]
    x += 6 * (torch.rand(b, v, generator=g, device="cuda") < 20 / v)     # a few tokens stand out
    x = torch.where(torch.rand(b, v, generator=g, device="cuda") < 0.01, float("-inf"), x)   # a grammar's mask
    s["logits"] = x.contiguous()
    s["u"] = torch.rand(b, generator=g, device="cuda")
    kinds = {"usual": [(0.6, 20, 0.95, 0.0)], "greedy": [(0.0, 0, 1.0, 0.0)], "free": [(1.0, 0, 1.0, 0.0)],
             "mixed": [(0.6, 20, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (0.8, 40, 1.0, 0.05), (1.3, 0, 0.9, 0.0),
                       (0.0, 0, 1.0, 0.0), (0.7, 1000, 0.8, 0.0), (1.0, 0, 1.0, 0.1)]}[case["settings"]]
    rows = [kinds[i % len(kinds)] for i in range(b)]
    for i, name in enumerate(("temperature", "top_k", "top_p", "min_p")):
        s[name] = torch.tensor([r[i] for r in rows], dtype=torch.int32 if name == "top_k" else torch.float32,
                               device="cuda")
    s["token"] = torch.zeros(b, dtype=torch.int32, device="cuda")
    s["logprob"] = torch.zeros(b, dtype=torch.float32, device="cuda")


# -------------------------------------------------------------------- runs
def run(s):
    c = s["case"]
    return {"attend": _run_attend, "append": _run_append, "evict": _run_evict, "sample": _run_sample}[c["op"]](s, c)


def _run_attend(s, c):
    if own:
        if c["accumulate"]:
            out = s["kv"].attend(s["q"], window=c["window"], acc=s["acc"], acc_out=s["acc_out"])
            return {"out": out, "acc": s["acc_out"]}
        return {"out": s["kv"].attend(s["q"], window=c["window"])}
    kv, dim = c["kv_heads"], c["dim"]
    batch, heads, _ = s["q"].shape
    stride = s["table"].shape[1] * c["page"]
    rows = torch.arange(c["longest"], device="cuda")
    pg, at = _address(s["table"], c["page"], rows)
    lens = s["lens"][:, None]
    seen = (rows[None] < lens) & (rows[None] >= lens - (c["window"] or stride))     # [b, rows]
    k = s["k"][pg, :, at[None]].float().transpose(1, 2)                               # [b, kv, rows, dim]
    v = torch.where(seen[:, None, :, None], s["v"][pg, :, at[None]].float().transpose(1, 2), 0.0)
    q = s["q"].reshape(batch, kv, heads // kv, dim)
    x = torch.where(seen[:, None, None], (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(dim)), float("-inf"))
    top = x.amax(3, keepdim=True)
    p = torch.where(seen[:, None, None], torch.exp(x - top), 0.0)
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = (p @ v).reshape(batch, heads, dim)
    if not c["accumulate"]:
        return {"out": out}
    w = p.sum(2)                                                                      # [b, kv, rows]
    old = s["acc"][..., :c["longest"]]
    new = torch.where(rows[None, None] == lens[:, None] - 1, w, old + w)
    acc = s["acc_out"].clone()
    acc[..., :c["longest"]] = torch.where(rows[None, None] < lens[:, None], new, acc[..., :c["longest"]])
    return {"out": out, "acc": acc}


def _rotated(x, w, pos):
    """RMSNorm over the head (w None: none), then the pairs (i, i + dim/2) turned by pos * base^(-2i/dim).  The angle
    is the one thing held in 64 bits: a position of 100000 in 32 bits would be off by a hundredth of a turn."""
    dim = x.shape[-1]
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    i = torch.arange(dim // 2, device="cuda", dtype=torch.float64)
    angle = (pos.double()[:, None] * _BASE ** (-2 * i / dim))[:, None]
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[..., :dim // 2], x[..., dim // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _run_append(s, c):
    if own:
        q = s["kv"].append(s["q"], s["key"], s["value"], s["pos"], freq_base=_BASE, q_norm=s["q_norm"],
                           k_norm=s["k_norm"], eps=_EPS, seq=s["seq"], row=s["row"], out=s["q_out"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    q = _rotated(s["q"], s["q_norm"], s["pos"])
    row, seq = s["row"].long(), s["seq"].long()
    pg = s["table"].long()[seq, row // c["page"]]
    s["k"][pg, :, row % c["page"]] = _rotated(s["key"], s["k_norm"], s["pos"]).to(s["k"].dtype)
    s["v"][pg, :, row % c["page"]] = s["value"].to(s["v"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _run_evict(s, c):
    if own:
        s["kv"].evict(s["acc"], s["pos"], s["next_pos"], c["budget"], n_recent=c["recent"], n_sink=c["sinks"],
                      acc_out=s["acc_out"], pos_out=s["pos_out"], lens_out=s["lens_out"])
        return {"k": s["k"], "v": s["v"], "acc": s["acc_out"], "pos": s["pos_out"], "lens": s["lens_out"]}
    batch, kv, stride = s["acc"].shape
    rows = torch.arange(stride, device="cuda")
    n = s["lens"].long()[:, None, None]
    left = torch.clamp(n, max=c["budget"])
    valid = rows < n
    kept_anyway = (s["pos"] >= s["next_pos"][:, None, None] - c["recent"]) | (s["pos"] < c["sinks"])
    kind = torch.where(valid, torch.where(kept_anyway, 2, 1), 0)
    weight = torch.where(torch.isnan(s["acc"]), float("-inf"), s["acc"])
    # by kind, then by weight, then the lowest row: two stable sorts, the lesser key first
    order = torch.argsort(weight, dim=2, descending=True, stable=True)
    order = order.gather(2, torch.argsort(kind.gather(2, order), dim=2, descending=True, stable=True))
    rank = torch.zeros_like(order).scatter_(2, order, rows.expand_as(order))
    kept = rank < left
    hole, mover = (rows < left) & ~kept, (rows >= left) & kept
    holes = torch.argsort(hole.to(torch.int8), dim=2, descending=True, stable=True)     # the holes, in order, first
    to = torch.where(mover, holes.gather(2, torch.clamp(torch.cumsum(mover, 2) - 1, min=0)), rows)
    source = rows.expand_as(to).clone().scatter_(2, torch.where(mover, to, stride - 1), torch.where(mover, rows, stride - 1))
    source = torch.where(hole, source, rows)                                             # row r is filled from source[r]
    acc, pos = s["acc"].gather(2, source), s["pos"].gather(2, source)
    b, j = torch.arange(batch, device="cuda")[:, None, None], torch.arange(kv, device="cuda")[None, :, None]
    table = s["table"].long()
    first = min(c["budget"], stride)
    src, dst = source[..., :first], rows[:first].expand(batch, kv, first)
    src, dst = (table[b, src // c["page"]], j, src % c["page"]), (table[b, dst // c["page"]], j, dst % c["page"])
    s["k"][dst] = s["k"][src]
    s["v"][dst] = s["v"][src]
    inside = rows < left
    return {"k": s["k"], "v": s["v"], "acc": torch.where(inside, acc, s["acc_out"]),
            "pos": torch.where(inside, pos, s["pos_out"]), "lens": left[:, 0, 0].to(torch.int32)}


def _part(of, total):
    """floor(of * total / 2^24), exactly, for of <= 2^24 and total < 2^62."""
    return (total >> 24) * of + (((total & 0xFFFFFF) * of) >> 24)


def _run_sample(s, c):
    if own:
        from styx_b200 import ops
        token, logprob = ops.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                                    token=s["token"], logprob=s["logprob"])
        return {"token": token, "logprob": logprob}
    x = torch.where(torch.isnan(s["logits"]), float("-inf"), s["logits"])
    v = x.shape[1]
    top = x.amax(1, keepdim=True)
    hot = s["temperature"][:, None] > 0
    y = torch.where(x == top, 0.0, (x - top) * (1.0 / s["temperature"][:, None]))
    w = torch.where(hot, torch.exp(y), (x == top).float()) * (top > float("-inf"))
    # sums of whole numbers: the same in any order
    weight = (w * 2.0 ** _UNIT).to(torch.int64)
    k = torch.where(s["top_k"] > 0, s["top_k"], v)[:, None]
    k = torch.where(hot, k, 1)
    order = torch.argsort(x, dim=1, descending=True, stable=True)
    sorted_weight = torch.where(torch.arange(v, device="cuda") < k, weight.gather(1, order), 0)
    so_far = torch.cumsum(sorted_weight, 1)
    p24 = torch.round(torch.clamp(s["top_p"], max=1.0) * 2.0 ** 24).to(torch.int64)[:, None]
    need = torch.clamp(_part(p24, so_far[:, -1:]), min=1)
    inside = (so_far - sorted_weight < need) & (w.gather(1, order) >= s["min_p"][:, None])
    kept = torch.zeros_like(weight).scatter_(1, order, torch.where(inside, sorted_weight, 0))
    so_far = torch.cumsum(kept, 1)
    total = so_far[:, -1:]
    u24 = torch.clamp((s["u"] * 2.0 ** 24).to(torch.int64), max=2 ** 24 - 1)[:, None]
    token = (so_far <= _part(u24, total)).sum(1, keepdim=True)
    some = total > 0
    logprob = y.gather(1, torch.clamp(token, max=v - 1)) - torch.log(total.float() * 2.0 ** -_UNIT)
    return {"token": torch.where(some, token, -1)[:, 0].to(torch.int32),
            "logprob": torch.where(some, logprob, float("-inf"))[:, 0]}


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "sample":
        # the logits once; an exponential, a comparison and a sum for each
        n = case["batch"] * case["vocab"]
        return {"bytes": 4 * n + 32 * case["batch"], "flops": 4 * n}
    size, kv, dim = _BYTES[case["type"]], case["kv_heads"], case["dim"]
    if op == "append":
        n, heads = case["tokens"], case["heads"]
        return {"bytes": n * dim * (4 * (2 * heads + 2 * kv) + 2 * kv * size) + 12 * n, "flops": n * (heads + kv) * dim * 6}
    lens = _lens(case)
    if op == "attend":
        rows = sum(min(n, case["window"] or n) for n in lens)
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": rows * kv * dim * 2 * size + case["batch"] * case["heads"] * dim * 8 + 4 * pages
                + (sum(lens) * kv * 8 if case["accumulate"] else 0),
                "flops": 4 * rows * case["heads"] * dim}
    left = [min(n, case["budget"]) for n in lens]
    # weights and positions read, those of the rows that stay written, and the rows that move, read and written:
    # where weights are spread evenly, the same share of the rows beyond the budget as of all
    moved = sum(m * (n - m) / n for n, m in zip(lens, left) if n)
    return {"bytes": kv * (8 * sum(lens) + 8 * sum(left) + moved * dim * size * 4), "flops": kv * sum(lens)}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict, "sample": _exact_sample}[
        case["op"]](s, case)


def _exact_attend(s, c):
    """Sequence by sequence, over its own rows alone."""
    kv, dim, page = c["kv_heads"], c["dim"], c["page"]
    gqa = c["heads"] // kv
    out = torch.zeros(c["batch"], c["heads"], dim, dtype=torch.float64, device="cuda")
    acc = s["acc_out"].double() if c["accumulate"] else None
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        first = max(0, n - c["window"]) if c["window"] else 0
        pages = s["table"][b, :-(-n // page)].tolist()
        for j in range(kv):
            k = torch.cat([s["k"][p, j] for p in pages])[first:n].double()
            v = torch.cat([s["v"][p, j] for p in pages])[first:n].double()
            p = torch.softmax(s["q"][b, j * gqa:(j + 1) * gqa].double() @ k.T / math.sqrt(dim), -1)
            out[b, j * gqa:(j + 1) * gqa] = p @ v
            if c["accumulate"]:
                acc[b, j, :n] = s["acc"][b, j, :n].double()
                acc[b, j, n - 1] = 0.0
                acc[b, j, first:n] += p.sum(0)
    return {"out": out, "acc": acc} if c["accumulate"] else {"out": out}


def _exact_append(s, c):
    n, dim, page = c["tokens"], c["dim"], c["page"]

    def turned(x, w):
        z = x.double()
        if w is not None:
            z = z / torch.sqrt(z.pow(2).sum(-1, keepdim=True) / dim + _EPS) * w.double()
        z = torch.complex(z[..., :dim // 2], z[..., dim // 2:])
        f = torch.tensor([_BASE ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device="cuda")
        a = s["pos"].double()[:, None, None] * f
        z = z * torch.polar(torch.ones_like(a), a)
        return torch.cat([z.real, z.imag], -1)

    k, v = s["k"].double(), s["v"].double()
    table, seq, row = s["table"].cpu().numpy(), s["seq"].cpu().numpy(), s["row"].cpu().numpy()
    at = torch.from_numpy(table[seq, row // page].astype(np.int64)).cuda()
    inner = torch.from_numpy((row % page).astype(np.int64)).cuda()
    heads = torch.arange(c["kv_heads"], device="cuda")
    k[at[:, None], heads[None], inner[:, None]] = turned(s["key"], s["k_norm"])
    v[at[:, None], heads[None], inner[:, None]] = s["value"].double()
    return {"q": turned(s["q"], s["q_norm"]), "k": k, "v": v}


def _exact_evict(s, c):
    k, v = s["k"].double().cpu().numpy(), s["v"].double().cpu().numpy()
    acc, pos = s["acc"].cpu().numpy(), s["pos"].cpu().numpy()
    table, lens, nxt = s["table"].cpu().numpy(), s["lens"].cpu().numpy(), s["next_pos"].cpu().numpy()
    out, page = np.zeros(acc.shape), c["page"]
    for b in range(c["batch"]):
        n = int(lens[b])
        left = min(n, c["budget"])
        for j in range(c["kv_heads"]):
            safe = (pos[b, j, :n] >= nxt[b] - c["recent"]) | (pos[b, j, :n] < c["sinks"])
            # lexsort: its last key counts first
            best = np.lexsort((np.arange(n), -acc[b, j, :n].astype(np.float64), ~safe))[:left]
            holes = np.setdiff1d(np.arange(left), best)
            movers = np.sort(best[best >= left])
            k[table[b, holes // page], j, holes % page] = k[table[b, movers // page], j, movers % page]
            v[table[b, holes // page], j, holes % page] = v[table[b, movers // page], j, movers % page]
            line = acc[b, j, :left].astype(np.float64)
            line[holes] = acc[b, j, movers]
            out[b, j, :left] = line
    return {"k": k, "v": v, "acc": out, "pos": None, "lens": None}


def _exact_sample(s, c):
    x = s["logits"].double().cpu().numpy()
    par = {n: s[n].double().cpu().numpy() for n in ("u", "temperature", "top_k", "top_p", "min_p")}
    logprob = np.full(c["batch"], -np.inf)
    for b in range(c["batch"]):
        t, top = par["temperature"][b], x[b].max()
        if t <= 0:
            logprob[b] = 0.0
            continue
        w = np.exp((x[b] - top) / t)
        order = np.argsort(-x[b], kind="stable")
        if par["top_k"][b] > 0:
            order = order[:int(par["top_k"][b])]
        cum = np.cumsum(w[order])
        order = order[(cum - w[order] < par["top_p"][b] * cum[-1]) & (w[order] >= par["min_p"][b])]
        order = np.sort(order)
        cum = np.cumsum(w[order])
        i = order[np.searchsorted(cum, par["u"][b] * cum[-1], side="right")]
        logprob[b] = (x[b, i] - top) / t - np.log(cum[-1])
    return {"token": None, "logprob": logprob}
