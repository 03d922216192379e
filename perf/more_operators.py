"""The operators of prompts in chunks over a paged KV cache: what is measured,
and their plain forms.

  plan     how many new tokens each sequence gets from what it wants, the
           token budget and the free pages; pages given and taken back; the
           sequence, row and position of every token
  append   per-head RMSNorm, rotary embedding (half or interleaved pairs, part
           of the head, scaled frequencies), K and V rows into the pages, q in
           the type that the attention takes
  attend   causal attention of the new tokens of every sequence over its pages

Pools are [n_pages][n_kv_heads][page_size][head_dim]; row r of sequence b is
in page table[b][r // page_size].  Tokens lie sequence after sequence, those of
sequence b are start[b] .. start[b + 1] - 1 and its last rows.  The plain forms
are elementary torch operations in 32 bits; with `own` the framework's calls
run instead.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6
_BASE = 1_000_000.0      # rotary base of the benchmark's decode step
_MOST = 32 * 8192 * 8192    # scores of the longest prompt: what a plain pass holds in 32 bits


# ------------------------------------------------------------------- cases
def _attend(name, batch, heads, kv_heads, dim, page, dtype, q_type, new, longest, lens, window=0):
    return {"name": name, "op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "type": dtype, "q_type": q_type, "new": new, "longest": longest, "lens": lens,
            "window": window}


def _append(name, seqs, tokens, heads, kv_heads, dim, page, dtype, q_type, longest, n_dims, pairs, scaling, norms=True):
    return {"name": name, "op": "append", "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "type": dtype, "q_type": q_type, "longest": longest, "n_dims": n_dims,
            "pairs": pairs, "scaling": scaling, "norms": norms}


def _plan(name, seqs, tokens, page, longest, kind):
    return {"name": name, "op": "plan", "seqs": seqs, "tokens": tokens, "page": page, "longest": longest,
            "kind": kind}


def listed():
    return [
        # the first message of one conversation: nothing but latency
        _attend("attend few tokens f16", 1, 32, 4, 128, 16, "f16", "f32", 5, 37, "even"),
        # drafted tokens of a full batch are checked: five a sequence, over caches of every age
        _attend("attend drafts bf16", 32, 32, 4, 128, 64, "bf16", "bf16", 5, 4096, "ragged"),
        # a whole prompt at once
        _attend("attend prompt f16", 1, 32, 4, 128, 64, "f16", "f16", 8192, 8192, "even"),
        # prompts of several requests, most with a prefix in the cache already, 16 query heads per kv head
        _attend("attend prompts ragged bf16", 8, 64, 4, 128, 64, "bf16", "bf16", 1021, 4099, "ragged"),
        # a late chunk of a whole book
        _attend("attend late chunk bf16", 1, 32, 4, 128, 64, "bf16", "bf16", 512, 131071, "even"),
        # the serving command's own types: f32 activations over f16 rows
        _attend("attend prompt f32 over f16", 1, 32, 4, 128, 64, "f16", "f32", 2048, 4096, "even"),
        # the cache in the activations' own type, as the single-sequence path keeps it; only a window is seen
        _attend("attend window f32", 4, 32, 4, 128, 32, "f32", "f32", 500, 4099, "ragged", window=1024),
        # one decode step of a full batch, half of each head turned
        _append("append step partial f16", 64, 64, 32, 4, 128, 64, "f16", "f16", 8192, 64, "interleaved", "none"),
        # prompts of several requests at positions beyond the trained length
        _append("append prompts yarn bf16", 6, 8191, 32, 4, 128, 64, "bf16", "bf16", 4000, 128, "half", "yarn"),
        # a decode step: one token each, now and then a page
        _plan("plan step", 64, 64, 64, 8192, "step"),
        # requests come and go: prompts wait for their turn, finished ones give their pages back
        _plan("plan admissions", 256, 16384, 16, 16384, "mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "plan"])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 4, 8])
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    q_type = "f32" if dtype == "f32" else rng.choice([dtype, dtype, "f32"])
    gqa = rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
    if op == "attend":
        batch = _log(rng, 1, 64)
        heads = gqa * kv_heads
        # the plain form's scores, products of f32 rows, and the pools bound the sizes
        most = _MOST // (8 if dtype == "f32" or dim == 256 else 1) // (batch * heads)
        longest = _log(rng, 1, min(131071, max(2, most // 4), max(2, 64 * 8192 * 4 * 128 // (batch * kv_heads * dim))))
        new = _log(rng, 1, max(1, min(longest, 8192, most // longest)))
        c = _attend("", batch, heads, kv_heads, dim, page, dtype, q_type, new, longest, rng.choice(["even", "ragged"]),
                    rng.choice([0, 0, 0, max(1, longest // 3)]))
    elif op == "append":
        seqs = _log(rng, 1, 64)
        tokens = seqs if rng.random() < 0.5 else _log(rng, seqs, 8192)
        gqa = min(gqa, 8)
        dim = min(dim, 128)
        c = _append("", seqs, tokens, gqa * kv_heads, kv_heads, dim, page, dtype, q_type,
                    -(-tokens // seqs) + _log(rng, 1, 2000), rng.choice([dim, dim, dim // 2, dim - 16]),
                    rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "yarn", "factors"]),
                    rng.random() < 0.7)
    else:
        seqs = _log(rng, 1, 1024)
        tokens = _log(rng, max(16, seqs), 16384)
        c = _plan("", seqs, tokens, page, max(page, _log(rng, 64, 16384)), rng.choice(["step", "mixed", "mixed"]))
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _lens(case):
    """(rows, new tokens) of each sequence: all alike, or rows in even steps up to the longest and chunks of between
    half and all of the most, the first slot empty where there are four or more."""
    b, longest, new = case["batch"], case["longest"], case["new"]
    if case["lens"] == "even":
        return [longest] * b, [new] * b
    rows = [max(1, longest * (i + 1) // b) for i in range(b)]
    news = [min(rows[i], max(1, new - (i * 7) % max(1, new // 2))) for i in range(b)]
    if b >= 4:
        rows[0] = news[0] = 0
    return rows, news


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(g, case, batch, rows):
    """K and V pools with a tenth more pages than the sequences need, and a table that hands them out in no order."""
    width = -(-rows // case["page"])
    n_pages = batch * width + batch * width // 10 + 1
    table = torch.randperm(n_pages, generator=g, device="cuda")[:batch * width].reshape(batch, width)
    shape = (n_pages, case["kv_heads"], case["page"], case["dim"])
    pools = []
    for _ in range(2):
        pool = torch.empty(shape, dtype=_TYPES[case["type"]], device="cuda")
        for at in range(0, n_pages, 4096):      # in parts: no second pool in 32 bits
            part = pool[at:at + 4096]
            part.copy_(_normal(g, *part.shape))
        pools.append(pool)
    return pools[0], pools[1], table.to(torch.int32).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": dict(case)}
    {"attend": _prepare_attend, "append": _prepare_append, "plan": _prepare_plan}[case["op"]](s, case, g)
    if own:
        # the objects that a server keeps for as long as it runs
        from styx_b200 import ops
        if case["op"] == "plan":
            s["planner"] = ops.PagedPlan(s["table"], case["page"], s["free"], case["tokens"])
        else:
            s["kv"] = ops.PagedKV(s["k"], s["v"], s["table"], s["lens"])
        if case["op"] == "append":
            s["rope"] = ops.Rope(case["n_dims"], _BASE, interleaved=case["pairs"] == "interleaved",
                                 scaling=case["scaling"] if case["scaling"] in ("linear", "yarn") else None,
                                 factor=_FACTOR, orig_ctx=_ORIG, factors=s["factors"])
    return s


def _prepare_attend(s, c, g):
    batch, heads, dim = c["batch"], c["heads"], c["dim"]
    s["k"], s["v"], s["table"] = _pool(g, c, batch, c["longest"])
    rows, news = _lens(c)
    order = torch.randperm(batch, generator=g, device="cuda")
    s["lens"] = _int(rows)[order].contiguous()
    new = _int(news)[order]
    s["start"] = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0, dtype=torch.int32)]).contiguous()
    n = sum(news)
    # heads of every sharpness: scores of spread 1/2 to 4
    sharp = torch.exp(torch.rand(heads, generator=g, device="cuda") * math.log(8.0)) / 2
    s["q"] = (_normal(g, n, heads, dim) * sharp[:, None]).to(_TYPES[c["q_type"]]).contiguous()
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(n, heads, device="cuda")
    # what lies past a sequence's end was never written, or anything else wrote it
    r = torch.arange(s["table"].shape[1] * c["page"], device="cuda")
    b, r = torch.nonzero(r[None] >= s["lens"][:, None], as_tuple=True)
    pg = s["table"].long()[b, r // c["page"]]
    s["k"][pg, :, r % c["page"]] = float("nan")
    s["v"][pg, :, r % c["page"]] = float("inf")


_FACTOR, _ORIG, _FAST, _SLOW = 4.0, 32768, 32.0, 1.0      # a context four times the trained one


def _prepare_append(s, c, g):
    n, seqs, heads, kv, dim = c["tokens"], c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    s["k"], s["v"], s["table"] = _pool(g, c, seqs, c["longest"])
    # q, k and v lie side by side, as one projection leaves them
    qkv = _normal(g, n, (heads + 2 * kv) * dim)
    s["q"], s["key"], s["value"] = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv * dim, kv * dim], 1))
    s["q_norm"] = torch.rand(dim, generator=g, device="cuda") + 0.5 if c["norms"] else None
    s["k_norm"] = torch.rand(dim, generator=g, device="cuda") + 0.5 if c["norms"] else None
    # what a model file divides its frequencies by
    s["factors"] = torch.exp2(torch.rand(c["n_dims"] // 2, generator=g, device="cuda") * 3) \
        if c["scaling"] == "factors" else None
    t = torch.arange(n, device="cuda")
    seq = t * seqs // n                                    # consecutive tokens of a prompt, prompt after prompt
    first = torch.searchsorted(seq, torch.arange(seqs, device="cuda"))
    count = torch.bincount(seq, minlength=seqs)
    before = torch.floor(torch.rand(seqs, generator=g, device="cuda") * (c["longest"] - count + 1)).long()
    s["seq"] = seq.to(torch.int32).contiguous()
    s["row"] = (before[seq] + t - first[seq]).to(torch.int32).contiguous()
    s["lens"] = (before + count).to(torch.int32).contiguous()
    # positions run ahead of rows where rows were evicted
    s["pos"] = (s["row"].long() + (torch.rand(seqs, generator=g, device="cuda") * 100000).long()[seq]).to(
        torch.int32).contiguous()
    s["q_out"] = torch.zeros(n, heads, dim, device="cuda", dtype=_TYPES[c["q_type"]])


def _prepare_plan(s, c, g):
    seqs, page = c["seqs"], c["page"]
    width = -(-c["longest"] // page)

    def some(lo, hi):                                      # spread over the logarithm
        return torch.exp(torch.rand(seqs, generator=g, device="cuda") * math.log((hi + 1) / lo)).mul(lo).floor().long()

    lens = torch.clamp(some(1, c["longest"]) - 1, max=width * page)
    held = -(-lens // page)
    if c["kind"] == "step":
        want = torch.ones_like(lens)
    else:
        kind = torch.rand(seqs, generator=g, device="cuda")
        lens = torch.where(kind < 0.2, 0, lens)            # done: its pages go back
        want = torch.where(kind < 0.2, 0, torch.where(kind < 0.6, 1, some(1, c["longest"])))
        lens = torch.where(kind > 0.9, lens // 2, lens)    # rows were evicted
    # of a pool that could hold every sequence at its longest, most pages are elsewhere: the last to come often find none
    used = int(held.sum())
    left = max(8, int(torch.rand((), generator=g, device="cuda") * (c["tokens"] // page + seqs)))
    n_pages = seqs * width + c["tokens"] // page + seqs + 8
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None] < held[:, None]
    s["table"][at] = ids[:used]
    s["free"] = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    s["free"][:left] = ids[used:used + left]
    s["n_free"] = _int([left])
    s["lens"], s["held"], s["want"] = (x.to(torch.int32).contiguous() for x in (lens, held, want))
    s["next_pos"] = (lens + some(1, 5000)).to(torch.int32).contiguous()


# -------------------------------------------------------------------- runs
def run(s):
    c = s["case"]
    return {"attend": _run_attend, "append": _run_append, "plan": _run_plan}[c["op"]](s, c)


def _run_attend(s, c):
    if own:
        out = s["kv"].attend_chunk(s["q"], s["start"], window=c["window"], out=s["out"], lse=s["lse"])
        return {"out": out, "lse": s["lse"]}
    n, heads, dim = s["q"].shape
    kv, page, batch, most = c["kv_heads"], c["page"], c["batch"], c["new"]
    start, lens = s["start"].long(), s["lens"].long()
    new = start[1:] - start[:-1]
    # every sequence's tokens as [batch, most]; those past its own are computed like its last and thrown away
    i = torch.arange(most, device="cuda")
    token = torch.clamp(torch.minimum(start[:-1, None] + i, start[1:, None] - 1), 0, n - 1)
    at = (lens - new)[:, None] + torch.minimum(i[None], new[:, None] - 1)                # [b, most]: rows of the tokens
    rows = torch.arange(c["longest"], device="cuda")
    pg, inner = s["table"].long()[:, rows // page], rows % page
    inside = (rows[None] < lens[:, None])[:, None, :, None]
    k = torch.where(inside, s["k"][pg, :, inner[None]].transpose(1, 2).float(), 0.0)     # [b, kv, rows, dim]
    v = torch.where(inside, s["v"][pg, :, inner[None]].transpose(1, 2).float(), 0.0)
    q = s["q"].float()[token].reshape(batch, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    seen = (rows <= at[..., None]) & (rows > at[..., None] - (c["window"] or c["longest"]))    # [b, most, rows]
    x = q.reshape(batch, kv, -1, dim) @ k.transpose(2, 3)
    x = x.reshape(batch, kv, heads // kv, most, c["longest"]).mul_(1.0 / math.sqrt(dim))
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = torch.clamp(x.amax(4, keepdim=True), min=-1e30)
    p = x.sub_(top).exp_()
    total = p.sum(4, keepdim=True)
    p = p.reshape(batch, kv, -1, c["longest"]) @ v
    p = p.reshape(batch, kv, heads // kv, most, dim) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(batch, most, heads)
    keep = i[None] < new[:, None]
    out = p.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)[keep]
    return {"out": out.to(s["q"].dtype), "lse": lse[keep]}


def _frequencies(c, factors):
    """(radians per position of every pair, what a turned pair is scaled by), in 64 bits."""
    n = c["n_dims"]
    i = torch.arange(n // 2, device="cuda", dtype=torch.float64)
    f = _BASE ** (-2 * i / n)
    if factors is not None:
        f = f / factors.double()
    if c["scaling"] == "linear":
        return f / _FACTOR, 1.0
    if c["scaling"] != "yarn":
        return f, 1.0
    lo = n * math.log(_ORIG / (_FAST * 2 * math.pi)) / (2 * math.log(_BASE))
    hi = n * math.log(_ORIG / (_SLOW * 2 * math.pi)) / (2 * math.log(_BASE))
    lo, hi = max(0, math.floor(lo)), min(n - 1, math.ceil(hi))
    ramp = torch.clamp((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
    return f * (1 - ramp) + f / _FACTOR * ramp, 1 + 0.1 * math.log(_FACTOR)


def _turned(c, x, w, pos, factors):
    """RMSNorm over the head (w None: none), then the pairs of the first n_dims elements turned.  The angle is the one
    thing held in 64 bits: a position of 100000 in 32 bits would be off by a hundredth of a turn."""
    n = c["n_dims"]
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    f, magnitude = _frequencies(c, factors)
    angle = (pos.double()[:, None] * f)[:, None]
    co, si = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * magnitude).float()
    if c["pairs"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * co - b * si, a * si + b * co, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * co - b * si, a * si + b * co], -1).flatten(-2), x[..., n:]], -1)


def _run_append(s, c):
    if own:
        q = s["kv"].append(s["q"], s["key"], s["value"], s["pos"], rope=s["rope"], q_norm=s["q_norm"],
                           k_norm=s["k_norm"], eps=_EPS, seq=s["seq"], row=s["row"], out=s["q_out"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    q = _turned(c, s["q"], s["q_norm"], s["pos"], s["factors"]).to(s["q_out"].dtype)
    row, seq = s["row"].long(), s["seq"].long()
    pg = s["table"].long()[seq, row // c["page"]]
    s["k"][pg, :, row % c["page"]] = _turned(c, s["key"], s["k_norm"], s["pos"], s["factors"]).to(s["k"].dtype)
    s["v"][pg, :, row % c["page"]] = s["value"].to(s["v"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _run_plan(s, c):
    if own:
        p = s["planner"].run(s["want"], s["lens"], s["held"], s["n_free"], s["next_pos"])
        return {"start": p.start, "seq": p.seq, "row": p.row, "pos": p.pos, "lens": p.lens, "held": p.held,
                "n_free": p.n_free, "next_pos": p.next_pos, "table": s["table"], "free": s["free"]}
    seqs, width = s["table"].shape
    page, tokens = c["page"], c["tokens"]
    lens, held = s["lens"].long(), s["held"].long()
    n_free = s["n_free"].long()
    want = torch.minimum(torch.clamp(s["want"].long(), min=0), width * page - lens)
    before = torch.cumsum(want, 0) - want
    t = torch.minimum(want, torch.clamp(tokens - before, min=0))
    target = (lens + t + page - 1) // page
    # pages that are not needed any more go on the stack, sequence after sequence
    at = torch.arange(width, device="cuda")
    back = (at[None] >= target[:, None]) & (at[None] < held[:, None])
    place = n_free + torch.cumsum(back.flatten(), 0).reshape(back.shape) - 1
    free = torch.cat([s["free"], s["free"][:1]])
    free.scatter_(0, torch.where(back, place, free.numel() - 1).flatten(), s["table"].flatten())
    top = n_free + back.sum()
    # and from its top come those that are
    need = torch.clamp(target - held, min=0)
    earlier = torch.cumsum(need, 0) - need
    got = torch.minimum(need, torch.clamp(top - earlier, min=0))
    number = torch.minimum(earlier, top)[:, None] + at[None] - held[:, None]
    comes = (at[None] >= held[:, None]) & (at[None] < (held + got)[:, None])
    popped = free[torch.clamp(top - 1 - number, 0, free.numel() - 1)]
    s["table"].copy_(torch.where(comes, popped, s["table"]))
    s["free"].copy_(free[:-1])
    granted = torch.minimum(t, torch.clamp((held + got) * page - lens, min=0))
    end = torch.cumsum(granted, 0)
    start = torch.cat([torch.zeros_like(end[:1]), end])
    i = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(end, i, right=True)
    real = seq < seqs
    seq = torch.clamp(seq, max=seqs - 1)
    nth = i - start[seq]
    int32 = torch.int32
    return {"start": start.to(int32), "seq": torch.where(real, seq, 0).to(int32),
            "row": torch.where(real, lens[seq] + nth, -1).to(int32),
            "pos": torch.where(real, s["next_pos"].long()[seq] + nth, 0).to(int32), "lens": (lens + granted).to(int32),
            "held": torch.where(held > target, target, held + got).to(int32), "n_free": (top - got.sum()).to(int32),
            "next_pos": (s["next_pos"] + granted).to(int32), "table": s["table"], "free": s["free"]}


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "plan":
        # per sequence five numbers in and four out, per token three out, per page that moves one in and one out
        n, tokens = case["seqs"], case["tokens"]
        return {"bytes": 36 * n + 12 * tokens + 8 * (tokens // case["page"]), "flops": 4 * n + 3 * tokens}
    size, q_size, kv, dim, heads = _BYTES[case["type"]], _BYTES[case["q_type"]], case["kv_heads"], case["dim"], case["heads"]
    if op == "append":
        n = case["tokens"]
        return {"bytes": n * dim * (4 * (heads + 2 * kv) + heads * q_size + 2 * kv * size) + 12 * n,
                "flops": n * (heads + kv) * dim * 6}
    rows, news = _lens(case)
    window = case["window"]
    cached = scores = 0
    for r, n in zip(rows, news):
        # token i of n sees min(r - n + i + 1, window) rows
        scores += sum(min(r - n + i + 1, window) for i in range(n)) if window else n * (r - n) + n * (n + 1) // 2
        cached += min(r, window + n - 1) if window and n else r if n else 0
    return {"bytes": cached * kv * dim * 2 * size + sum(news) * heads * (2 * dim * q_size + 4),
            "flops": 4 * scores * heads * dim}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "plan":
        return None                        # whole numbers
    s = prepare(case, seed)
    return _exact_attend(s, case) if case["op"] == "attend" else _exact_append(s, case)


def _exact_attend(s, c):
    """Sequence by sequence, head by head, some tokens at a time, over the rows that there are alone."""
    page, gqa, dim = c["page"], c["heads"] // c["kv_heads"], c["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    start, lens, table = s["start"].tolist(), s["lens"].tolist(), s["table"].tolist()
    for b, n in enumerate(lens):
        lo, hi = start[b], start[b + 1]
        pages = table[b][:-(-n // page)]
        for j in range(c["kv_heads"] if hi > lo else 0):
            k = torch.cat([s["k"][p, j] for p in pages])[:n].double()
            v = torch.cat([s["v"][p, j] for p in pages])[:n].double()
            for h in range(j * gqa, (j + 1) * gqa):
                for t0 in range(lo, hi, 2048):
                    t1 = min(hi, t0 + 2048)
                    row = torch.arange(n - hi + t0, n - hi + t1, device="cuda")[:, None]
                    r = torch.arange(n, device="cuda")[None]
                    hidden = (r > row) | (r <= row - c["window"]) if c["window"] else r > row
                    x = (s["q"][t0:t1, h].double() @ k.T / math.sqrt(dim)).masked_fill_(hidden, -math.inf)
                    lse[t0:t1, h] = torch.logsumexp(x, 1)
                    out[t0:t1, h] = torch.softmax(x, 1) @ v
    return {"out": out, "lse": lse}


def _exact_append(s, c):
    n, page, heads = c["n_dims"], c["page"], torch.arange(c["kv_heads"], device="cuda")
    f, magnitude = [], 1.0
    for i in range(n // 2):
        w = _BASE ** (-2.0 * i / n)
        if s["factors"] is not None:
            w /= float(s["factors"][i])
        if c["scaling"] == "linear":
            w /= _FACTOR
        if c["scaling"] == "yarn":
            # turns over the trained length: more than _FAST are kept as they are, fewer than _SLOW are stretched
            edge = [n * math.log(_ORIG / (turns * 2 * math.pi)) / (2 * math.log(_BASE)) for turns in (_FAST, _SLOW)]
            lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), n - 1)
            part = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w * (1.0 - part) + w * part / _FACTOR
            magnitude = 0.1 * math.log(_FACTOR) + 1.0
        f.append(w)
    a = s["pos"].double()[:, None, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(a, magnitude), a)

    def turned(x, w):
        z = x.double()
        if w is not None:
            z = z / torch.sqrt(z.pow(2).sum(-1, keepdim=True) / c["dim"] + _EPS) * w.double()
        if c["pairs"] == "half":
            y = torch.complex(z[..., :n // 2], z[..., n // 2:n]) * turn
            return torch.cat([y.real, y.imag, z[..., n:]], -1)
        y = torch.view_as_complex(z[..., :n].unflatten(-1, (-1, 2)).contiguous()) * turn
        return torch.cat([torch.view_as_real(y).flatten(-2), z[..., n:]], -1)

    k, v = s["k"].double(), s["v"].double()
    row = s["row"].long()
    at = torch.gather(s["table"][s["seq"].long()].long(), 1, (row // page)[:, None])
    k[at, heads[None], (row % page)[:, None]] = turned(s["key"], s["k_norm"])
    v[at, heads[None], (row % page)[:, None]] = s["value"].double()
    return {"q": turned(s["q"], s["q_norm"]), "k": k, "v": v}
