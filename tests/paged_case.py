"""Paged KV caches for the tests, and the operators' definitions in 64 bits
(numpy), sequence by sequence."""
import numpy as np
import torch

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make_cache(rng, lens, n_kv, hd, page, dtype, spare=3, max_rows=None, gap=0):
    """(PagedKV, k rows, v rows) with the rows of every sequence as float64
    arrays [n][n_kv][hd]; what no sequence uses holds NaN.  gap: elements
    between the pages of the pools."""
    from styx_b200 import ops
    lens = list(lens)
    width = max(1, -(-max(list(lens) + [max_rows or 0]) // page))
    n_pages = len(lens) * width + spare
    t = TYPES[dtype]
    size = n_kv * page * hd + gap
    pools = []
    for _ in range(2):
        flat = torch.full((n_pages, size), float("nan"), dtype=t, device=DEV)
        pools.append(flat[:, :n_kv * page * hd].unflatten(1, (n_kv, page, hd)))
    k, v = pools
    table = torch.from_numpy(rng.permutation(n_pages)[:len(lens) * width].reshape(len(lens), width).astype(np.int32))
    ks, vs = [], []
    for b, n in enumerate(lens):
        kb = torch.from_numpy(rng.normal(0, 1, (n, n_kv, hd)).astype(np.float32)).to(t)
        vb = torch.from_numpy(rng.normal(0, 1, (n, n_kv, hd)).astype(np.float32)).to(t)
        for p in range(-(-n // page)):
            lo, hi = p * page, min(n, (p + 1) * page)
            k[int(table[b, p]), :, :hi - lo] = kb[lo:hi].transpose(0, 1).to(DEV)
            v[int(table[b, p]), :, :hi - lo] = vb[lo:hi].transpose(0, 1).to(DEV)
        ks.append(kb.double().numpy())
        vs.append(vb.double().numpy())
    kv = ops.PagedKV(k, v, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    return kv, ks, vs


def read_rows(kv, b, n):
    """Rows 0..n-1 of sequence b of both pools, float64 [n][n_kv][hd]."""
    page = kv.k.shape[2]
    out = []
    for pool in (kv.k, kv.v):
        rows = [pool[int(p)].transpose(0, 1) for p in kv.table[b, :-(-n // page)].tolist()]
        out.append(torch.cat(rows)[:n].double().cpu().numpy() if n else np.zeros((0,)))
    return out


def attend_ref(q, ks, vs, scale, window=0):
    """(out [B][H][hd], lse [B][H], weights: per sequence [n_kv][n])"""
    B, H, hd = q.shape
    out, lse, ws = np.zeros((B, H, hd)), np.full((B, H), -np.inf), []
    for b in range(B):
        n = ks[b].shape[0]
        n_kv = ks[b].shape[1]
        first = max(0, n - window) if window else 0
        w = np.zeros((n_kv, n))
        for h in range(H if n else 0):
            j = h // (H // n_kv)
            s = ks[b][first:, j] @ q[b, h].astype(np.float64) * scale
            e = np.exp(s - s.max())
            p = e / e.sum()
            out[b, h] = p @ vs[b][first:, j]
            lse[b, h] = s.max() + np.log(e.sum())
            w[j, first:] += p
        ws.append(w)
    return out, lse, ws


def rope_norm_ref(x, w, pos, base, eps):
    """x [n][heads][hd] float64"""
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    th = pos.astype(np.float64)[:, None, None] * base ** (-2.0 * np.arange(hd // 2) / hd)
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([a * np.cos(th) - b * np.sin(th), a * np.sin(th) + b * np.cos(th)], -1)


def evict_ref(acc, pos, n, next_pos, budget, n_recent, n_sink):
    """src[r], r < min(n, budget): the row whose content ends in row r."""
    left = min(n, budget)
    safe = (pos[:n] >= next_pos - n_recent) | (pos[:n] < n_sink)
    a = np.where(np.isnan(acc[:n]), -np.inf, acc[:n]).astype(np.float64)
    order = sorted(range(n), key=lambda r: (not safe[r], -a[r] if not safe[r] else 0.0, r))
    stay = set(order[:left])
    src = list(range(left))
    places = [r for r in range(left) if r not in stay]
    movers = [r for r in range(left, n) if r in stay]
    assert len(places) == len(movers)
    for p, m in zip(places, movers):
        src[p] = m
    return np.array(src, dtype=np.int64)
