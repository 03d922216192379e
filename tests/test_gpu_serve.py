"""Batched decoding over a paged KV cache on the GPU (include/styx_serve.h)
against the operators' definitions in 64 bits (tests/paged_case.py).

Tolerances, from the arithmetic: attention 1e-5 of max|out| (the bound of
the single-sequence attention: scores of size ~10 rounded to f32 move a
weight by ~1e-6, sums of some thousand rows add as much again); accumulated
weights the same, relative to a weight sum of 1 per head.  Rotated q 2e-6 of
max|q| (an RMSNorm, a rounded sine and cosine, three roundings: 6 x 2^-24
and a margin); K and V rows half an ulp of the cache's type more.  Eviction
moves whole rows and sampling sums whole numbers: equal.  A drawn token's
interval of the 64-bit cumulative distribution may miss u by 3e-6: a weight
exp(y) carries |y| x 2^-23 + 2^-22 of relative error, averaged over the
distribution at most 10 x 2^-23 + 2^-22, and 2^-40 for each of the tokens.
"""
import numpy as np
import pytest
import torch

from styx_b200 import StyxError, _lib, ops
from tests.paged_case import (DEV, TYPES, attend_ref, evict_ref, make_cache, read_rows, rope_norm_ref)

pytestmark = pytest.mark.gpu


def T(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def close(got, exp, tol, what=""):
    got, exp = np.asarray(got, np.float64), np.asarray(exp, np.float64)
    assert got.shape == exp.shape and np.all(np.isfinite(got)), what
    err = np.max(np.abs(got - exp), initial=0.0) / max(np.max(np.abs(exp), initial=0.0), 1e-30)
    assert err <= tol, f"{what} {err:.2e} > {tol}"


def queries(rng, b, h, hd):
    return (rng.normal(0, 1, (b, h, hd)) * rng.uniform(0.3, 3, (1, h, 1))).astype(np.float32)


# ------------------------------------------------------------------ attention
CASES = [
    # lens, heads, kv heads, head_dim, page, type, window
    ([1], 32, 4, 128, 16, "f16", 0),
    ([37], 32, 4, 128, 16, "bf16", 0),
    ([0, 1, 15, 16, 17, 31, 32, 33], 32, 4, 128, 16, "f16", 0),
    ([0, 0], 8, 2, 64, 64, "bf16", 0),
    ([700, 3, 0, 129, 64], 64, 4, 128, 64, "bf16", 0),
    ([700, 3, 0, 129, 64], 64, 4, 128, 64, "f32", 0),
    ([2049, 513], 32, 4, 128, 32, "f16", 300),
    ([300, 20, 1], 16, 2, 128, 256, "f32", 17),
    ([100, 7], 6, 6, 64, 16, "f16", 0),
    ([257, 90], 28, 4, 80, 16, "bf16", 0),
    ([130, 61], 5, 1, 96, 32, "f16", 1),
    ([66, 400], 14, 2, 256, 16, "bf16", 0),
    ([66, 400], 14, 2, 256, 16, "f32", 0),
    ([70], 40, 1, 120, 64, "f16", 0),
    ([70, 90], 33, 1, 8, 64, "bf16", 0),
    ([50], 4, 4, 4, 1, "f32", 0),
    ([45, 99], 8, 4, 128, 1, "f16", 50),
    ([45, 99], 8, 4, 128, 2, "bf16", 0),
    ([5000], 16, 8, 64, 4096, "f16", 0),
    ([16384], 8, 1, 128, 128, "bf16", 0),
]


@pytest.mark.parametrize("lens,heads,n_kv,hd,page,dtype,window", CASES)
def test_attend(lens, heads, n_kv, hd, page, dtype, window):
    rng = np.random.default_rng(sum(lens) + heads + hd)
    kv, ks, vs = make_cache(rng, lens, n_kv, hd, page, dtype)
    q = queries(rng, len(lens), heads, hd)
    out, lse, _ = attend_ref(q, ks, vs, hd ** -0.5, window)
    l = torch.zeros(len(lens), heads, device=DEV)
    got = kv.attend(T(q), window=window, lse=l).cpu().numpy()
    close(got, out, 1e-5)
    l = l.cpu().numpy()
    assert np.array_equal(np.isinf(l), np.isinf(lse))
    fine = np.isfinite(lse)
    assert np.max(np.abs(l[fine] - lse[fine]), initial=0) < 1e-5 * max(1, np.max(np.abs(lse[fine]), initial=0))
    kv.ctx.check_device_error()
    again = kv.attend(T(q), window=window).cpu().numpy()
    assert np.array_equal(got, again)          # the same bits, call after call


@pytest.mark.parametrize("lens,heads,n_kv,hd,page,dtype,window", CASES)
def test_attend_accumulates_the_weights(lens, heads, n_kv, hd, page, dtype, window):
    rng = np.random.default_rng(sum(lens) + heads + hd + 1)
    kv, ks, vs = make_cache(rng, lens, n_kv, hd, page, dtype)
    q = queries(rng, len(lens), heads, hd)
    out, _, ws = attend_ref(q, ks, vs, hd ** -0.5, window)
    stride = kv.max_rows + 5
    acc = rng.uniform(0, 2, (len(lens), n_kv, stride)).astype(np.float32)
    exp = np.full((len(lens), n_kv, stride), 7.0)
    for b, n in enumerate(lens):
        exp[b, :, :n] = acc[b, :, :n] + ws[b]
        if n:
            exp[b, :, n - 1] = ws[b][:, n - 1]      # the newest row enters with its own weight
            acc[b, :, n - 1] = np.nan
        acc[b, :, n:] = np.nan
    acc_out = torch.full((len(lens), n_kv, stride), 7.0, device=DEV)
    got = kv.attend(T(q), window=window, acc=T(acc), acc_out=acc_out)
    close(got.cpu().numpy(), out, 1e-5)
    got_acc = acc_out.cpu().numpy()
    assert np.all(np.isfinite(got_acc))
    assert np.max(np.abs(got_acc - exp)) < 1e-5 * heads / n_kv
    inplace = T(acc)
    kv.attend(T(q), window=window, acc=inplace)
    for b, n in enumerate(lens):
        assert np.array_equal(inplace.cpu().numpy()[b, :, :n], got_acc[b, :, :n])
    kv.ctx.check_device_error()


def test_attend_sharp_and_flat_heads():
    """One row with all the weight (scores of +-200: every other weight
    underflows), equal rows (the mean of V), scores all far below zero."""
    rng = np.random.default_rng(4)
    for dtype in TYPES:
        kv, ks, vs = make_cache(rng, [333, 333], 2, 128, 32, dtype)
        q = np.zeros((2, 16, 128), np.float32)
        for h in range(8):
            q[0, h] = ks[0][40 * h, 0] * 20.0            # row 40 h by far
            q[1, h] = -ks[1][40 * h, 0] * 20.0
        out, lse, _ = attend_ref(q, ks, vs, 128 ** -0.5)
        got = kv.attend(T(q)).cpu().numpy()
        # scores up to 230 in f32: 2^-24 x 230 x 4 of a weight
        close(got, out, 6e-5, dtype)
        close(got[:, 8:], np.stack([np.broadcast_to(v[:, 1].mean(0), (8, 128)) for v in vs]), 1e-5, dtype)


def test_attend_last_page_next_to_another_sequences_rows():
    """A page past the sequence's end belongs to somebody else, or to nobody."""
    rng = np.random.default_rng(5)
    kv, ks, vs = make_cache(rng, [50, 64], 2, 64, 16, "f16", max_rows=200)
    kv.table[0, 4:] = -7
    kv.table[1, 4:] = 1 << 30
    q = queries(rng, 2, 8, 64)
    close(kv.attend(T(q)).cpu().numpy(), attend_ref(q, ks, vs, 0.125)[0], 1e-5)
    kv.ctx.check_device_error()


def test_attend_page_outside_the_pool_is_skipped_and_reported():
    rng = np.random.default_rng(6)
    for bad in (-1, 1 << 20):
        kv, ks, vs = make_cache(rng, [50, 64], 2, 64, 16, "bf16")
        kv.table[0, 1] = bad
        q = queries(rng, 2, 8, 64)
        got = kv.attend(T(q)).cpu().numpy()
        with pytest.raises(StyxError):
            kv.ctx.check_device_error()
        ks[0], vs[0] = (np.delete(a, range(16, 32), 0) for a in (ks[0], vs[0]))
        close(got, attend_ref(q, ks, vs, 0.125)[0], 1e-5)
        kv.ctx.check_device_error()


def test_attend_length_outside_the_table_is_clamped_and_reported():
    rng = np.random.default_rng(7)
    kv, ks, vs = make_cache(rng, [32, 32], 1, 64, 16, "f16")
    q = queries(rng, 2, 4, 64)
    exp = kv.attend(T(q)).cpu().numpy()
    kv.lens.copy_(torch.tensor([33, 32]))
    got = kv.attend(T(q)).cpu().numpy()
    with pytest.raises(StyxError):
        kv.ctx.check_device_error()
    assert np.array_equal(got, exp)
    kv.lens.copy_(torch.tensor([32, -1]))
    got = kv.attend(T(q)).cpu().numpy()
    with pytest.raises(StyxError):
        kv.ctx.check_device_error()
    assert np.array_equal(got[0], exp[0]) and not got[1].any()


def test_attend_pools_of_more_than_2_31_elements():
    """Pages of one layer far apart: element offsets past 32 bits."""
    rng = np.random.default_rng(8)
    far = (1 << 30) + 64
    flat = [torch.empty(2 * far + 2 * 16 * 64, dtype=torch.float16, device=DEV) for _ in range(2)]
    k, v = (f.as_strided((3, 2, 16, 64), (far, 16 * 64, 64, 1)) for f in flat)
    for t in (k, v):
        t.copy_(T(rng.normal(0, 1, (3, 2, 16, 64)).astype(np.float16)))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    kv = ops.PagedKV(k, v, table, torch.tensor([41], dtype=torch.int32, device=DEV))
    ks, vs = ([a] for a in read_rows(kv, 0, 41))
    q = queries(rng, 1, 4, 64)
    close(kv.attend(T(q)).cpu().numpy(), attend_ref(q, ks, vs, 0.125)[0], 1e-5)
    pos = torch.tensor([[9000] + list(range(1, 48))] * 2, dtype=torch.int32, device=DEV)[None].contiguous()
    acc = torch.arange(96, dtype=torch.float32, device=DEV).reshape(1, 2, 48).contiguous()
    kv.evict(acc, pos, torch.tensor([48], dtype=torch.int32, device=DEV), 20)
    new = read_rows(kv, 0, 20)
    src = evict_ref(acc[0, 0].cpu().numpy(), pos[0, 0].cpu().numpy(), 41, 48, 20, 0, 0)
    assert np.array_equal(new[0][:, 0], ks[0][src, 0]) and np.array_equal(new[1][:, 1], vs[0][src, 1])
    kv.append(None, torch.ones(1, 2, 64, device=DEV), torch.ones(1, 2, 64, device=DEV),
              torch.zeros(1, dtype=torch.int32, device=DEV), 1e4, row=torch.tensor([9], dtype=torch.int32, device=DEV))
    assert read_rows(kv, 0, 20)[1][9].min() == 1.0
    kv.ctx.check_device_error()


def test_attend_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(9)
    kv, ks, vs = make_cache(rng, [200, 77], 4, 128, 16, "f16")
    q = T(queries(rng, 2, 32, 128))
    exp = kv.attend(q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = kv.attend(q, stream=s)
    s.synchronize()
    assert torch.equal(got, exp)
    out = torch.zeros_like(exp)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.attend(q, out=out)
    for lens in ([200, 77], [13, 0], [1, 200 - 56]):
        kv.lens.copy_(torch.tensor(lens))
        g.replay()
        torch.cuda.synchronize()
        ref = attend_ref(q.cpu().numpy(), [ks[0][:lens[0]], ks[1][:min(77, lens[1])]],
                         [vs[0][:lens[0]], vs[1][:min(77, lens[1])]], 128 ** -0.5)[0]
        close(out.cpu().numpy()[0], ref[0], 1e-5)
        if lens[1] <= 77:
            close(out.cpu().numpy()[1], ref[1], 1e-5)


# --------------------------------------------------------------------- append
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.mark.parametrize("n_seqs,n_tokens,heads,n_kv,hd,page,dtype,norms",
                         [(1, 1, 32, 4, 128, 16, "f16", True), (5, 5, 8, 2, 64, 64, "bf16", True),
                          (3, 77, 5, 1, 96, 16, "f32", True), (2, 300, 4, 4, 256, 32, "f16", False),
                          (64, 64, 32, 4, 128, 64, "bf16", True), (4, 9, 7, 7, 8, 1, "bf16", False),
                          (2, 33, 0, 2, 80, 128, "f16", True), (1, 1000, 16, 2, 128, 256, "f32", True),
                          (3, 3, 3, 1, 4, 2, "f32", True)])
def test_append(n_seqs, n_tokens, heads, n_kv, hd, page, dtype, norms):
    rng = np.random.default_rng(n_tokens + hd)
    count = -(-n_tokens // n_seqs)
    kv, ks, vs = make_cache(rng, [count + 40] * n_seqs, n_kv, hd, page, dtype)
    seq = np.arange(n_tokens) % n_seqs
    row = rng.permutation(count + 40)[: count].astype(np.int32)[np.arange(n_tokens) // n_seqs]
    pos = rng.integers(0, 200000, n_tokens).astype(np.int32)
    qkv = rng.normal(0, 2, (n_tokens, (heads + 2 * n_kv) * hd + 3)).astype(np.float32)
    d = T(qkv)
    cut = lambda a, lo, n: a[:, lo * hd:(lo + n) * hd].reshape(n_tokens, n, hd)   # noqa: E731
    sl = lambda lo, n: d[:, lo * hd:(lo + n) * hd].unflatten(1, (n, hd))          # noqa: E731
    qn, kn = ((rng.uniform(0.5, 1.5, hd).astype(np.float32) if norms else None) for _ in range(2))
    q_out = kv.append(sl(0, heads) if heads else None, sl(heads, n_kv), sl(heads + n_kv, n_kv), T(pos), 1e6,
                      q_norm=T(qn) if norms else None, k_norm=T(kn) if norms else None, eps=1e-6,
                      seq=T(seq.astype(np.int32)), row=T(row))
    kv.ctx.check_device_error()
    if heads:
        exp = rope_norm_ref(cut(qkv, 0, heads).astype(np.float64), qn, pos, 1e6, 1e-6)
        close(q_out.cpu().numpy(), exp, 2e-6)
    ek = rope_norm_ref(cut(qkv, heads, n_kv).astype(np.float64), kn, pos, 1e6, 1e-6)
    ev = cut(qkv, heads + n_kv, n_kv).astype(np.float64)
    for t in range(n_tokens):
        ks[seq[t]][row[t]], vs[seq[t]][row[t]] = ek[t], ev[t]
    for b in range(n_seqs):
        gk, gv = read_rows(kv, b, count + 40)
        top = np.max(np.abs(ks[b]))
        assert np.all(np.abs(gk - ks[b]) <= HALF_ULP[dtype] * np.abs(ks[b]) + 2e-6 * top + 2.0 ** -25)
        assert np.all(np.abs(gv - vs[b]) <= HALF_ULP[dtype] * np.abs(vs[b]) + 2.0 ** -25)


def test_append_default_rows_and_empty_slots():
    """row None: lens - 1; a slot of length 0 and a negative row write nothing and give a zero q."""
    rng = np.random.default_rng(11)
    kv, ks, vs = make_cache(rng, [5, 0, 17], 2, 64, 16, "f16", max_rows=32)
    before = [read_rows(kv, b, 32) for b in range(3)]
    x = rng.normal(0, 1, (3, 8, 64)).astype(np.float32)
    pos = np.array([4, 99, 16], np.int32)
    q = kv.append(T(x), T(x[:, :2]), T(x[:, 2:4]), T(pos), 1e4)
    kv.ctx.check_device_error()
    exp = rope_norm_ref(x.astype(np.float64), None, pos, 1e4, 0)
    exp[1] = 0
    close(q.cpu().numpy(), exp, 2e-6)
    for b, r in ((0, 4), (1, None), (2, 16)):
        now = read_rows(kv, b, 32)
        for i, ref in ((0, exp[b, :2]), (1, x[b, 2:4])):
            same = np.ones(32, bool)
            if r is not None:
                same[r] = False
                assert np.max(np.abs(now[i][r] - ref)) <= 2.0 ** -11 * np.max(np.abs(ref)) + 1e-6
            assert np.array_equal(now[i][same], before[b][i][same], equal_nan=True)
    q = kv.append(T(x), T(x[:, :2]), T(x[:, 2:4]), T(pos), 1e4, row=torch.tensor([-1, -5, -1], dtype=torch.int32, device=DEV))
    assert not q.any()
    kv.ctx.check_device_error()


def test_append_out_of_range_is_skipped_and_reported():
    rng = np.random.default_rng(12)
    for kind in ("row", "seq", "page"):
        kv, ks, vs = make_cache(rng, [5, 9], 2, 64, 16, "f16")
        seq, row = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([2, 3], dtype=torch.int32)
        if kind == "row":
            row[0] = 16
        elif kind == "seq":
            seq[0] = 2
        else:
            kv.table[0, 0] = 99
        pools = [kv.k.clone(), kv.v.clone()]
        x = T(rng.normal(0, 1, (2, 2, 64)).astype(np.float32))
        kv.append(x, x, x, torch.tensor([0, 0], dtype=torch.int32, device=DEV), 1e4, seq=seq.to(DEV), row=row.to(DEV))
        with pytest.raises(StyxError):
            kv.ctx.check_device_error()
        changed = (kv.k != pools[0]) & ~torch.isnan(kv.k)
        assert {int(i) for i in changed.nonzero()[:, 0]} == {int(kv.table[1, 0])}


def test_append_attend_agree_with_the_single_sequence_path():
    """The step of the flat f32 cache (styx_qk_norm_rope_kv, styx_attn_decode)
    and the same step over pages: 2e-6 of max, 1e-5 after the attention."""
    rng = np.random.default_rng(13)
    nh, nkv, hd, n = 32, 4, 128, 300
    kv, ks, vs = make_cache(rng, [n], nkv, hd, 16, "f32")
    kc = T(np.concatenate(ks).reshape(n, -1).astype(np.float32))
    vc = T(np.concatenate(vs).reshape(n, -1).astype(np.float32))
    q, k, v = (T(rng.normal(0, 1, (1, h, hd)).astype(np.float32)) for h in (nh, nkv, nkv))
    w = T(rng.uniform(0.5, 1.5, hd).astype(np.float32))
    pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    q2, k2 = q.clone(), k.clone()
    ops.qk_norm_rope_kv(q2, k2, v, w, w, 1e-6, nh, nkv, hd, 1e6, pos, kc, vc, n)
    flat = ops.attn_decode(q2.reshape(-1), kc, vc, n, hd, nkv * hd, nh // nkv, hd ** -0.5).reshape(1, nh, hd)
    q3 = kv.append(q, k, v, pos, 1e6, q_norm=w, k_norm=w)
    close(q3.cpu().numpy(), q2.cpu().numpy(), 2e-6)
    close(kv.attend(q3).cpu().numpy(), flat.cpu().numpy(), 1e-5)


# ------------------------------------------------------------------- eviction
@pytest.mark.parametrize("lens,n_kv,hd,page,dtype,budget,recent,sink,kind",
                         [([40], 2, 64, 16, "f16", 16, 4, 2, "plain"),
                          ([40, 3, 0, 16, 17], 2, 64, 16, "bf16", 16, 4, 2, "ties"),
                          ([1], 1, 8, 1, "f16", 1, 0, 0, "plain"), ([2], 1, 4, 1, "f32", 1, 1, 0, "plain"),
                          ([1000, 999], 4, 128, 64, "f16", 999, 100, 4, "ties"),
                          ([1000, 5], 1, 96, 32, "f32", 1, 0, 0, "plain"),
                          ([5000, 1025, 1024], 2, 64, 256, "bf16", 1024, 512, 4, "special"),
                          ([300], 3, 80, 16, "f16", 128, 128, 0, "same"),
                          ([300, 300], 3, 80, 16, "f16", 128, 0, 0, "same"),
                          ([20000], 1, 8, 64, "f16", 7001, 50, 1, "ties"),
                          ([70000], 1, 8, 64, "f16", 64, 8, 4, "plain"), ([9000], 2, 8, 64, "f16", 4096, 0, 0, "magnitudes"),
                          ([3000, 4097], 2, 8, 32, "f16", 2500, 2400, 4, "plain"),
                          ([400000, 5], 1, 8, 64, "f16", 300000, 1000, 4, "ties")])
def test_evict(lens, n_kv, hd, page, dtype, budget, recent, sink, kind):
    rng = np.random.default_rng(sum(lens) + budget)
    kv, ks, vs = make_cache(rng, lens, n_kv, hd, page, dtype)
    B, stride = len(lens), kv.max_rows + 3
    acc = rng.exponential(1, (B, n_kv, stride)).astype(np.float32)
    if kind == "ties":
        acc = np.floor(acc * 3).astype(np.float32)
    elif kind == "same":
        acc[:] = 0.25
    elif kind == "magnitudes":      # every exponent there is, subnormal weights among them
        acc = np.exp2(rng.uniform(-149, 127, acc.shape)).astype(np.float32) * np.where(rng.uniform(size=acc.shape) < 0.1, -1, 1)
        acc = acc.astype(np.float32)
    elif kind == "special":
        which = rng.integers(0, 8, acc.shape)
        for i, x in enumerate((np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5)):
            acc[which == i] = x
    pos = np.stack([[rng.permutation(stride) for _ in range(n_kv)] for _ in range(B)]).astype(np.int32)
    nxt = np.array([stride - 2] * B, np.int32)
    acc_out = torch.full((B, n_kv, stride), 7.0, device=DEV)
    pos_out = torch.full((B, n_kv, stride), 7, dtype=torch.int32, device=DEV)
    lens_out = torch.zeros(B, dtype=torch.int32, device=DEV)
    a, p = T(acc), T(pos)
    for _ in range(2):      # the call repeats: the inputs are left as they are
        kv.evict(a, p, T(nxt), budget, recent, sink, acc_out=acc_out, pos_out=pos_out, lens_out=lens_out)
        kv.ctx.check_device_error()
        assert np.array_equal(lens_out.cpu().numpy(), np.minimum(lens, budget))
        ao, po = acc_out.cpu().numpy(), pos_out.cpu().numpy()
        for b, n in enumerate(lens):
            left = min(n, budget)
            gk, gv = read_rows(kv, b, left)
            for j in range(n_kv):
                src = evict_ref(acc[b, j], pos[b, j], n, int(nxt[b]), budget, recent, sink)
                assert np.array_equal(ao[b, j, :left], acc[b, j, src], equal_nan=True)
                assert np.array_equal(po[b, j, :left], pos[b, j, src])
                assert np.all(ao[b, j, left:] == 7) and np.all(po[b, j, left:] == 7)
                if left:
                    assert np.array_equal(gk[:, j], ks[b][src, j]) and np.array_equal(gv[:, j], vs[b][src, j])
        assert np.array_equal(a.cpu().numpy(), acc, equal_nan=True) and np.array_equal(p.cpu().numpy(), pos)


def test_evict_duplicate_positions_still_keep_the_budget():
    """More protected rows than the budget (positions that repeat): the lowest rows of them."""
    rng = np.random.default_rng(21)
    kv, ks, vs = make_cache(rng, [50], 1, 64, 16, "f16")
    acc = rng.uniform(0, 1, (1, 1, 64)).astype(np.float32)
    pos = np.full((1, 1, 64), 9, np.int32)
    _, _, n = kv.evict(T(acc), T(pos), T(np.array([10], np.int32)), 20, 5, 0)
    assert n.tolist() == [20]
    gk, _ = read_rows(kv, 0, 20)
    assert np.array_equal(gk, ks[0][:20])


def test_evict_then_decode_matches_attention_over_the_rows_that_stayed():
    rng = np.random.default_rng(22)
    kv, ks, vs = make_cache(rng, [400, 90], 2, 128, 16, "bf16")
    acc = rng.exponential(1, (2, 2, kv.max_rows)).astype(np.float32)
    pos = np.broadcast_to(np.arange(kv.max_rows, dtype=np.int32), acc.shape)
    a, p, n = kv.evict(T(acc), T(pos), T(np.array([400, 90], np.int32)), 128, 32, 4)
    kv.lens = n
    q = queries(rng, 2, 8, 128)
    got = kv.attend(T(q)).cpu().numpy()
    for b, rows in ((0, 400), (1, 90)):
        for j in range(2):
            src = evict_ref(acc[b, j], pos[b, j], rows, rows, 128, 32, 4)
            ref = attend_ref(q[b:b + 1, 4 * j:4 * j + 4], [ks[b][src][:, j:j + 1]], [vs[b][src][:, j:j + 1]], 128 ** -0.5)[0]
            close(got[b, 4 * j:4 * j + 4], ref[0], 1e-5)


# ------------------------------------------------------------------- sampling
def sample_ok(x, u, t, k, p, m, token, logprob):
    """The token's interval of the 64-bit distribution holds u, to 3e-6; its log-probability to 1e-5."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        assert token == -1 and logprob == -np.inf
        return
    if t <= 0:
        assert token == int(np.argmax(x)) and logprob == 0
        return
    with np.errstate(invalid="ignore"):
        y = np.where(x == top, 0.0, (x - top) / t)
    w = np.exp(y)
    order = np.argsort(-x, kind="stable")
    if k > 0:
        order = order[:k]
    cum = np.cumsum(w[order])
    tol = 3e-6
    lo, hi, lps = [], [], []    # with the fewest and the most tokens that the rounded sums may keep
    for kept in (order[(cum - w[order] < (min(p, 1.0) - tol) * cum[-1]) & (w[order] >= m * (1 + 1e-5))],
                 order[(cum - w[order] <= (min(p, 1.0) + tol) * cum[-1]) & (w[order] >= m * (1 - 1e-5))]):
        kept = np.sort(kept) if kept.size else order[:1]
        c = np.cumsum(w[kept])
        at = np.searchsorted(kept, token)
        if at < kept.size and kept[at] == token:
            lo.append((c[at] - w[token]) / c[-1])
            hi.append(c[at] / c[-1])
            lps.append(y[token] - np.log(c[-1]))
    assert lo, f"token {token} is not among those kept"
    near = 1e-5 * max(1, abs(lps[0])) + 2 * tol / max(min(p, 1.0), 1e-3)
    assert min(lps) - near <= logprob <= max(lps) + near, (lps, logprob)
    assert min(lo) - tol <= u <= max(hi) + tol, (u, lo, hi)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (0.8, 40, 1.0, 0.05), (1.3, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0),
            (0.7, 1000, 0.8, 0.0), (1.0, 0, 1.0, 0.1), (2.0, 1, 0.5, 0.5), (1.0, 10 ** 6, 0.999, 1e-6),
            (0.05, 0, 0.01, 0.0), (1.0, 3, 1.0, 1.0), (5.0, 0, 0.5, 0.0), (-1.0, 5, 0.3, 0.2), (1.0, -4, 2.0, -1.0)]


@pytest.mark.parametrize("vocab,rows,kind", [(1, 3, "plain"), (2, 5, "plain"), (31, 14, "plain"), (1000, 28, "plain"),
                                             (1000, 28, "ties"), (4097, 28, "mask"), (151936, 14, "plain"),
                                             (151936, 14, "ties"), (151936, 14, "flat"), (33333, 28, "low"),
                                             (200003, 14, "mask"), (262145, 5, "flat"), (65537, 28, "nan")])
def test_sample(vocab, rows, kind):
    rng = np.random.default_rng(vocab + rows)
    x = (rng.normal(0, 3, (rows, vocab))).astype(np.float32)
    if kind == "ties":
        x = np.round(x).astype(np.float32)
    elif kind == "flat":
        x[:] = 1.5
    elif kind == "mask":
        x[rng.uniform(size=x.shape) < 0.9] = -np.inf
    elif kind == "low":       # a mask of the type's lowest value
        x[rng.uniform(size=x.shape) < 0.9] = np.finfo(np.float32).min
    elif kind == "nan":
        x[rng.uniform(size=x.shape) < 0.3] = np.nan
        x[rng.uniform(size=x.shape) < 0.1] = -0.0
        x[rng.uniform(size=x.shape) < 0.1] = 0.0
    par = [SETTINGS[i % len(SETTINGS)] for i in range(rows)]
    u = rng.uniform(0, 1, rows).astype(np.float32)
    u[0] = 0.0
    u[-1] = np.float32(1 - 2.0 ** -24)
    t, k, p, m = (np.array([q[i] for q in par], np.int32 if i == 1 else np.float32) for i in range(4))
    token, logprob = ops.sample(T(x), T(u), T(t), T(k), T(p), T(m))
    token, logprob = token.cpu().numpy(), logprob.cpu().numpy()
    for b in range(rows):
        assert 0 <= token[b] < vocab
        sample_ok(x[b], float(u[b]), float(t[b]), int(k[b]), float(p[b]), min(float(m[b]), 1.0), int(token[b]),
                  float(logprob[b]))


def test_sample_rows_with_nothing_left_and_infinities():
    v = 5000
    x = np.full((6, v), -np.inf, np.float32)
    x[1, 77] = -3e38                       # one finite value
    x[2] = np.nan
    x[3, [5, 900]] = np.inf                # infinite logits share all the weight
    x[4] = np.finfo(np.float32).min        # all at the type's lowest value: uniform
    x[5, :] = 0
    x[5, 1000:] = -np.inf
    u = np.array([0.3, 0.9, 0.5, 0.75, 0.5, 0.9995], np.float32)
    token, lp = ops.sample(T(x), T(u))
    assert token.tolist() == [-1, 77, -1, 900, 2500, 999]
    exp = [-np.inf, 0.0, -np.inf, np.log(0.5), -np.log(v), -np.log(1000)]
    assert np.allclose(lp.cpu().numpy(), exp, rtol=1e-6, atol=1e-7)
    token, _ = ops.sample(T(x), T(u), temperature=torch.zeros(6, device=DEV))
    assert token.tolist() == [-1, 77, -1, 5, 0, 0]


def test_sample_ties_at_the_threshold_go_to_the_lowest_index():
    x = np.zeros((64, 3000), np.float32)
    x[:, 2000] = 1.0
    u = (np.arange(64, dtype=np.float32) + 0.5) / 64
    token, _ = ops.sample(T(x), T(u), top_k=torch.full((64,), 3, dtype=torch.int32, device=DEV))
    assert set(token.tolist()) == {0, 1, 2000}
    w = np.exp(-1.0)
    token, _ = ops.sample(T(x), T(u), top_p=torch.full((64,), (1 + 1.5 * w) / (1 + 2999 * w), device=DEV))
    assert set(token.tolist()) == {0, 1, 2000}


def test_sample_strides_defaults_and_streams():
    rng = np.random.default_rng(31)
    big = T(rng.normal(0, 2, (9, 4000)).astype(np.float32))
    u = T(rng.uniform(0, 1, 9).astype(np.float32))
    for view in (big[:, 1:3998], big[:, 3:4], big[::2, 7:1000]):
        n = view.shape[0]
        exp = ops.sample(view.contiguous(), u[:n].contiguous())
        got = ops.sample(view, u[:n].contiguous())
        assert torch.equal(exp[0], got[0]) and torch.equal(exp[1], got[1])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = ops.sample(view, u[:n].contiguous(), stream=s)
        s.synchronize()
        assert torch.equal(exp[0], got[0])


def test_sample_frequencies_follow_the_distribution():
    """20000 draws of 8 tokens: every frequency within five standard deviations."""
    p = np.array([0.4, 0.2, 0.15, 0.1, 0.06, 0.05, 0.03, 0.01])
    n = 20000
    x = T(np.broadcast_to(np.log(p), (n, 8)).astype(np.float32))
    u = T(np.random.default_rng(32).uniform(0, 1, n).astype(np.float32))
    token, lp = ops.sample(x, u)
    got = np.bincount(token.cpu().numpy(), minlength=8) / n
    assert np.all(np.abs(got - p) < 5 * np.sqrt(p * (1 - p) / n))
    assert np.allclose(lp.cpu().numpy(), np.log(p)[token.cpu().numpy()], atol=1e-6)


# ------------------------------------------------------------------- refusals
def test_refusals():
    rng = np.random.default_rng(41)
    kv, _, _ = make_cache(rng, [20, 30], 2, 64, 16, "f16")
    q = T(queries(rng, 2, 8, 64))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)   # noqa: E731
    f = lambda *s: torch.zeros(*s, device=DEV)                        # noqa: E731
    for call in (lambda: kv.attend(q[:1]), lambda: kv.attend(q.half()), lambda: kv.attend(q.transpose(0, 1)),
                 lambda: kv.attend(q.cpu()), lambda: kv.attend(q, acc_out=f(2, 2, 32)),
                 lambda: kv.attend(q, out=f(2, 8, 63)), lambda: kv.append(q, q, q, i32(0, 0), 1e4),
                 lambda: kv.append(q, q[:, :2].half(), q[:, :2], i32(0, 0), 1e4),
                 lambda: kv.append(q, q[:, :2], q[:, :2], f(2), 1e4),
                 lambda: ops.sample(f(3), f(3)), lambda: ops.sample(f(3, 4), f(2)),
                 lambda: ops.sample(f(4, 3).t(), f(3)), lambda: ops.sample(f(3, 4), f(3), top_k=f(3)),
                 lambda: ops.PagedKV(kv.k, kv.v, kv.table.long(), kv.lens),
                 lambda: ops.PagedKV(kv.k, kv.v.float(), kv.table, kv.lens),
                 lambda: ops.PagedKV(kv.k.transpose(1, 2), kv.v.transpose(1, 2), kv.table, kv.lens),
                 lambda: ops.PagedKV(kv.k, kv.v, kv.table, kv.lens[:1])):
        with pytest.raises(ValueError):
            call()
    acc, pos = f(2, 2, 32), torch.zeros(2, 2, 32, dtype=torch.int32, device=DEV)
    odd = lambda n_kv, page, hd, t=torch.float16: ops.PagedKV(   # noqa: E731
        torch.zeros(8, n_kv, page, hd, dtype=t, device=DEV), torch.zeros(8, n_kv, page, hd, dtype=t, device=DEV),
        kv.table, kv.lens)
    for call in (lambda: kv.attend(T(queries(rng, 2, 7, 64))),                      # not a multiple of n_kv_heads
                 lambda: kv.attend(q, window=-1), lambda: kv.attend(q, scale=float("nan")),
                 lambda: kv.attend(q, acc=f(2, 2, 31)),                             # shorter than the rows
                 lambda: odd(2, 24, 64).attend(q),                                  # page not a power of two
                 lambda: odd(2, 16, 12).attend(f(2, 8, 12)),                        # rows of 24 bytes
                 lambda: odd(2, 16, 264).attend(f(2, 8, 264)),
                 lambda: odd(2, 16, 2, torch.float32).attend(f(2, 8, 2)),
                 lambda: kv.append(q, q[:, :2], q[:, :2], i32(0, 0), 0.0),
                 lambda: kv.append(q, q[:, :2], q[:, :2], i32(0, 0), 1e4, out=q),   # in place
                 lambda: kv.append(f(3, 8, 64), f(3, 2, 64), f(3, 2, 64), i32(0, 0, 0), 1e4),   # 3 tokens, 2 sequences
                 lambda: kv.evict(acc, pos, i32(9, 9), 0), lambda: kv.evict(acc, pos, i32(9, 9), 8, 6, 3),
                 lambda: kv.evict(acc, pos, i32(9, 9), 8, -1),
                 lambda: kv.evict(acc, pos, i32(9, 9), 8, acc_out=acc),
                 lambda: kv.evict(acc, pos, i32(9, 9), 8, lens_out=kv.lens),
                 lambda: kv.evict(f(2, 2, 31), pos[..., :31].contiguous(), i32(9, 9), 8)):
        with pytest.raises(StyxError) as e:
            call()
        assert e.value.code == _lib.STYX_EINVAL
    L, cx = _lib.lib(), kv.ctx.handle
    assert L.styx_sample(cx, None, None, 4, 1, 4, None, None, None, None, None, None, None) == _lib.STYX_EINVAL
    assert L.styx_paged_attend(cx, None, None, 8, None, 1.0, 0, None, None, None, None, 0, None, 0) == _lib.STYX_EINVAL
    kv.attend(q)
    ws = torch.zeros(1 << 22, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(q)
    assert L.styx_paged_attend(cx, None, kv._ref, 8, q.data_ptr(), 1.0, 0, out.data_ptr(), None, None, None, 0,
                               ws.data_ptr(), 16) == _lib.STYX_EINVAL and b"workspace" in L.styx_last_error()
    kv.ctx.check_device_error()


@pytest.mark.parametrize("rows", [33, 130, 600])
def test_sample_rows_do_not_depend_on_their_batch(rows):
    """Batches of more rows than fit the device at once are taken in another order: the same tokens and logprobs, bit
    for bit, as eight rows at a time."""
    rng = np.random.default_rng(rows)
    V = 1000
    x = T(rng.normal(0, 3, (rows, V)).astype(np.float32))
    par = [SETTINGS[i % len(SETTINGS)] for i in rng.permutation(rows)]
    t, k, p, m = (T(np.array([q[i] for q in par], np.int32 if i == 1 else np.float32)) for i in range(4))
    u = T(rng.uniform(0, 1, rows).astype(np.float32))
    token, logprob = ops.sample(x, u, t, k, p, m)
    for i in range(0, rows, 8):
        s = slice(i, i + 8)
        tok, lp = ops.sample(x[s], u[s], t[s], k[s], p[s], m[s])
        assert torch.equal(tok, token[s]) and torch.equal(lp, logprob[s])


@pytest.mark.parametrize("vocab", [2049, 2100, 3000, 4096, 20000])
def test_sample_many_flat_rows(vocab):
    """More equal logits than one CTA sorts, few of them outside the first CTA's slice or all slices full: the
    threshold by bisection of the key (its sums share slots with the counts that chose it).  Whole numbers of equal
    weight: the token is exact."""
    rows = 300
    rng = np.random.default_rng(vocab)
    x = torch.zeros(rows, vocab, device=DEV)
    u24 = rng.integers(0, 1 << 24, rows)
    u = T((u24 / 2.0 ** 24).astype(np.float32))
    frac = rng.integers(1, 1 << 24, rows)                      # top-p as a fraction of 2^24
    ks = rng.integers(121, vocab, rows)
    one = 1 << 40
    kept_p = [-(-max(1, (vocab * one * int(f)) >> 24) // one) for f in frac]
    for _ in range(10):
        for kept, kw in ((kept_p, dict(top_p=T((frac / 2.0 ** 24).astype(np.float32)))),
                         (ks.tolist(), dict(top_k=T(ks.astype(np.int32))))):
            token, lp = ops.sample(x, u, **kw)
            exp = [((n * one * int(a)) >> 24) // one for n, a in zip(kept, u24)]
            assert token.tolist() == exp
            assert np.allclose(lp.cpu().numpy(), -np.log(np.array(kept)), atol=1e-5)
    ops.ctx(0).check_device_error()


# more segments than SMs: every warp (or pair of warps) of the tensor-core form has a share of its own
MANY = [
    # sequences, longest, heads, kv heads, head_dim, page, type, window
    (50, 400, 32, 4, 128, 16, "bf16", 0),
    (50, 400, 32, 4, 128, 64, "f16", 100),
    (40, 700, 64, 4, 128, 32, "bf16", 0),
    (160, 90, 12, 1, 64, 16, "f16", 0),
    (100, 300, 10, 2, 72, 64, "bf16", 33),
    (90, 260, 40, 2, 120, 16, "f16", 0),
    (200, 128, 8, 1, 128, 64, "f16", 0),
    (200, 300, 3, 1, 8, 16, "bf16", 0),
]


@pytest.mark.parametrize("n_seqs,longest,heads,n_kv,hd,page,dtype,window", MANY)
def test_attend_many_sequences(n_seqs, longest, heads, n_kv, hd, page, dtype, window):
    rng = np.random.default_rng(n_seqs + hd + heads)
    lens = rng.integers(0, longest + 1, n_seqs)
    lens[:6] = [0, 1, 16, 17, longest, longest - 1]
    lens = [int(n) for n in lens]
    test_attend(lens, heads, n_kv, hd, page, dtype, window)
    test_attend_accumulates_the_weights(lens, heads, n_kv, hd, page, dtype, window)


def test_attend_one_long_among_many_short():
    """A segment cut over many warps beside segments that are whole."""
    lens = [3] * 60 + [9000] + [0] * 20 + [40] * 80
    test_attend(lens, 16, 2, 128, 64, "bf16", 0)
    test_attend(lens, 16, 1, 128, 16, "f16", 0)


def test_attend_many_with_a_page_outside_the_pool():
    rng = np.random.default_rng(6)
    lens = [100] * 90
    kv, ks, vs = make_cache(rng, lens, 2, 128, 16, "f16")
    kv.table[7, 2] = 1 << 30                    # rows 32 to 47 of sequence 7
    q = queries(rng, 90, 16, 128)
    ks[7], vs[7] = np.delete(ks[7], range(32, 48), 0), np.delete(vs[7], range(32, 48), 0)
    out = attend_ref(q, ks, vs, 128 ** -0.5)[0]
    close(kv.attend(T(q)).cpu().numpy(), out, 1e-5)
    with pytest.raises(StyxError):
        kv.ctx.check_device_error()


def test_caches_of_one_shape_share_workspaces():
    rng = np.random.default_rng(8)
    a, ka, va = make_cache(rng, [40, 9], 2, 64, 16, "f16")
    b, kb, vb = make_cache(rng, [21, 33], 2, 64, 16, "f16")
    other, _, _ = make_cache(rng, [21, 33], 2, 64, 16, "bf16")
    b.share_workspaces(a)
    q = queries(rng, 2, 8, 64)
    for kv, ks, vs in ((a, ka, va), (b, kb, vb), (a, ka, va)):
        close(kv.attend(T(q)).cpu().numpy(), attend_ref(q, ks, vs, 0.125)[0], 1e-5)
    with pytest.raises(ValueError, match="share_workspaces"):
        other.share_workspaces(a)


@pytest.mark.parametrize("lens,heads,n_kv,hd,page,dtype", [([40, 9], 16, 2, 128, 16, "f16"), ([40, 9], 16, 2, 128, 16, "bf16"),
                                                            ([40, 9], 16, 2, 128, 16, "f32"), ([700, 33], 32, 2, 64, 64, "bf16"),
                                                            ([5000, 9], 8, 1, 128, 64, "f16"), ([5000, 9], 8, 1, 128, 64, "f32"),
                                                            ([300] * 90, 16, 2, 128, 64, "f16"), ([300] * 90, 32, 2, 72, 64, "bf16"),
                                                            ([60, 9], 8, 2, 256, 16, "f16")])
def test_attend_nan_and_infinite_scores_are_not_hidden(lens, heads, n_kv, hd, page, dtype):
    """The softmax over a NaN or a score of +inf is NaN, not the zeros of a sequence without rows: in q of one head,
    and in one row of K (all heads of its kv head).  The other heads and sequences keep their values (not their bits:
    the heads of a group move their maxima together)."""
    rng = np.random.default_rng(50)
    kv, _, _ = make_cache(rng, lens, n_kv, hd, page, dtype)
    q = T(queries(rng, len(lens), heads, hd))
    lse = torch.zeros(len(lens), heads, device=DEV)
    acc = torch.zeros(len(lens), n_kv, kv.max_rows, device=DEV)
    exp, exp_lse = kv.attend(q, lse=lse, acc=acc).clone(), lse.clone()
    exp_acc = acc.clone()

    def check(hit):                       # hit: [sequences][heads], True where NaN is expected
        got = kv.attend(q, lse=lse, acc=acc)
        assert torch.isnan(got[hit]).all() and torch.isnan(lse[hit]).all()
        close(got[~hit].cpu().numpy(), exp[~hit].cpu().numpy(), 2e-5)          # 1e-5 each
        assert (lse[~hit] - exp_lse[~hit]).abs().max() <= 2e-5 * max(1, exp_lse[~hit].abs().max().item())
        by_kv = hit.unflatten(1, (n_kv, -1)).any(2)
        for b, n in enumerate(lens):
            for j in range(n_kv):
                if by_kv[b, j]:
                    assert torch.isnan(acc[b, j, :n]).all()
                else:
                    assert (acc[b, j, :n] - exp_acc[b, j, :n]).abs().max() <= 2e-5 * heads / n_kv

    for bad in (float("nan"), float("inf")):
        hit = torch.zeros(len(lens), heads, dtype=torch.bool, device=DEV)
        hit[0, 3] = True
        keep = q[0, 3, 5].item()
        q[0, 3, 5] = bad
        acc.zero_()
        check(hit)
        q[0, 3, 5] = keep
    page_id, row = int(kv.table[0, 0]), 1
    kv.k[page_id, 0, row, 2] = float("nan")
    hit = torch.zeros(len(lens), heads, dtype=torch.bool, device=DEV)
    hit[0, :heads // n_kv] = True
    acc.zero_()
    check(hit)
    kv.ctx.check_device_error()


@pytest.mark.parametrize("budget", [48, 49, 2 ** 31 - 1])
def test_evict_with_a_budget_beyond_the_rows(budget):
    rng = np.random.default_rng(23)
    kv, ks, vs = make_cache(rng, [48, 7, 0], 2, 64, 16, "f16")
    acc, pos = rng.uniform(0, 1, (3, 2, 48)).astype(np.float32), rng.permutation(288).reshape(3, 2, 48).astype(np.int32)
    a, p, n = kv.evict(T(acc), T(pos), T(np.array([300, 300, 300], np.int32)), budget, 20, 4)
    kv.ctx.check_device_error()
    assert n.tolist() == [48, 7, 0]
    for b, m in enumerate([48, 7, 0]):
        assert np.array_equal(a[b, :, :m].cpu().numpy(), acc[b, :, :m]) and np.array_equal(p[b, :, :m].cpu().numpy(), pos[b, :, :m])
        gk, gv = read_rows(kv, b, m)
        assert m == 0 or (np.array_equal(gk, ks[b]) and np.array_equal(gv, vs[b]))


def test_append_refuses_a_q_out_over_k_or_v():
    """k and v are read by other warps than those that write q_out."""
    rng = np.random.default_rng(42)
    kv, _, _ = make_cache(rng, [20, 30], 2, 64, 16, "f16")
    buf = T(rng.normal(0, 1, 2 * 8 * 64 + 2 * 2 * 64).astype(np.float32))
    q, other = T(queries(rng, 2, 8, 64)), T(rng.normal(0, 1, (2, 2, 64)).astype(np.float32))
    pos = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    out = buf[:1024].view(2, 8, 64)
    for at in (0, 64, 1024 - 4):                              # its start, inside, its last 16 bytes
        over = buf[at:at + 256].view(2, 2, 64)
        for k, v in ((over, other), (other, over)):
            with pytest.raises(StyxError, match="overlaps") as e:
                kv.append(q, k, v, pos, 1e4, out=out)
            assert e.value.code == _lib.STYX_EINVAL
    exp = kv.append(q, other, other, pos, 1e4)
    assert torch.equal(kv.append(q, buf[1024:].view(2, 2, 64), other, pos, 1e4, out=out), exp)   # beside it
    kv.ctx.check_device_error()


def test_attend_refuses_weights_and_outputs_that_overlap_in_part():
    """acc_out may be acc and out may be q, row for row; shifted against each other a block would read what another has
    written."""
    rng = np.random.default_rng(43)
    kv, _, _ = make_cache(rng, [20, 30], 2, 64, 16, "f16")
    q = T(queries(rng, 2, 8, 64))
    acc = torch.zeros(2 * 2 * 32 + 8, device=DEV)
    line = lambda at: acc[at:at + 128].view(2, 2, 32)        # noqa: E731
    buf = torch.zeros(1024 + 64, device=DEV)
    at = lambda i: buf[i:i + 1024].view(2, 8, 64)            # noqa: E731
    at(0).copy_(q)
    for call in (lambda: kv.attend(q, acc=line(0), acc_out=line(4)), lambda: kv.attend(q, acc=line(4), acc_out=line(0)),
                 lambda: kv.attend(at(0), out=at(64)), lambda: kv.attend(at(64), out=at(0))):
        with pytest.raises(StyxError, match="overlap") as e:
            call()
        assert e.value.code == _lib.STYX_EINVAL
    exp = kv.attend(q)
    assert torch.equal(kv.attend(at(0), out=at(0)), exp)
    kv.ctx.check_device_error()


def test_evict_refuses_outputs_over_any_input_or_each_other():
    rng = np.random.default_rng(44)
    kv, _, _ = make_cache(rng, [20, 30], 2, 64, 16, "f16")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)   # noqa: E731
    acc, pos, nxt = torch.rand(2, 2, 32, device=DEV), torch.zeros(2, 2, 32, dtype=torch.int32, device=DEV), i32(40, 40)
    f = lambda t: t.view(torch.float32)                               # noqa: E731
    i = lambda t: t.view(torch.int32)                                 # noqa: E731
    out = torch.zeros(2, 2, 32, device=DEV)
    for kw in (dict(acc_out=f(pos)), dict(pos_out=i(acc)), dict(acc_out=out, pos_out=i(out)), dict(lens_out=nxt),
               dict(lens_out=pos.view(-1)[6:8]), dict(lens_out=i(acc).view(-1)[:2]), dict(lens_out=i(out).view(-1)[2:4], acc_out=out),
               dict(lens_out=i(out).view(-1)[2:4], pos_out=i(out))):
        with pytest.raises(StyxError, match="other arrays") as e:
            kv.evict(acc, pos, nxt, 8, **kw)
        assert e.value.code == _lib.STYX_EINVAL
    kv.ctx.check_device_error()


def test_sizes_of_one_have_no_stride():
    """One kv head, one page or one row a page: the strides of such a dimension say nothing about the layout."""
    rng = np.random.default_rng(45)
    lens = torch.tensor([3], dtype=torch.int32, device=DEV)
    for n_pages, n_kv, page in ((4, 1, 16), (1, 2, 16), (4, 2, 1), (1, 1, 16), (1, 1, 4), (4, 1, 1)):
        rows = min(3, n_pages * page)
        lens.fill_(rows)
        pool = [T(rng.normal(0, 1, (n_pages, n_kv, page, 64)).astype(np.float32)) for _ in range(2)]
        table = torch.arange(n_pages, dtype=torch.int32, device=DEV)[None]
        q = T(queries(rng, 1, 4, 64))
        exp = ops.PagedKV(*pool, table, lens).attend(q)
        size, dense = (n_pages, n_kv, page, 64), (n_kv * page * 64, page * 64, 64, 1)
        odd = tuple(7777 if n == 1 else s for n, s in zip(size, dense))
        k, v = pool[0].as_strided(size, odd), pool[1].as_strided(size, dense)
        t = table.as_strided((1, n_pages), (1, 1 if n_pages > 1 else 55))
        assert torch.equal(ops.PagedKV(k, v, t, lens).attend(q), exp)
    x = T(rng.normal(0, 1, (5, 1)).astype(np.float32))
    token, lp = ops.sample(x.as_strided((5, 1), (1, 9)), torch.zeros(5, device=DEV))
    assert token.tolist() == [0] * 5 and lp.tolist() == [0.0] * 5


# ------------------------------------------------------------ shapes that the tests above do not reach
@pytest.mark.parametrize("vocab,rows,kind", [(262145, 14, "plain"), (300001, 14, "ties"), (270000, 14, "mask"),
                                             (270001, 14, "low"), (400000, 14, "nan"), (1 << 20, 7, "plain")])
def test_sample_vocabularies_beyond_a_cluster(vocab, rows, kind):
    """One CTA per row and radix selection, on ordinary rows: every setting, ties at the threshold, masks, NaN."""
    test_sample(vocab, rows, kind)


def test_sample_beyond_a_cluster_draws_what_the_cluster_draws():
    """The same rows with and without a tail of -inf that no filter keeps: one token, one logprob (sums of whole
    numbers do not depend on the form)."""
    rng = np.random.default_rng(51)
    rows, v = 28, 200000
    x = np.round(rng.normal(0, 3, (rows, v)) * 4).astype(np.float32) / 4
    par = [SETTINGS[i % len(SETTINGS)] for i in range(rows)]
    t, k, p, m = (T(np.array([q[i] for q in par], np.int32 if i == 1 else np.float32)) for i in range(4))
    u = T(rng.uniform(0, 1, rows).astype(np.float32))
    a = ops.sample(T(x), u, t, k, p, m)
    b = ops.sample(T(np.concatenate([x, np.full((rows, 70000), -np.inf, np.float32)], 1)), u, t, k, p, m)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("hd,heads,n_kv", [(128, 9, 3), (12, 5, 1), (64, 4, 4)])
def test_append_with_one_norm_alone(hd, heads, n_kv, which):
    rng = np.random.default_rng(52)
    kv, _, _ = make_cache(rng, [9, 30, 31], n_kv, hd, 16, "f32")
    q, k, v = (rng.normal(0, 2, (3, h, hd)).astype(np.float32) for h in (heads, n_kv, n_kv))
    w, pos = rng.uniform(0.5, 1.5, hd).astype(np.float32), np.array([8, 29, 100000], np.int32)
    qn, kn = (w, None) if which == "q" else (None, w)
    got = kv.append(T(q), T(k), T(v), T(pos), 1e4, q_norm=None if qn is None else T(qn), k_norm=None if kn is None else T(kn))
    close(got.cpu().numpy(), rope_norm_ref(q.astype(np.float64), qn, pos, 1e4, 1e-6), 2e-6)
    ek = rope_norm_ref(k.astype(np.float64), kn, pos, 1e4, 1e-6)
    for b, r in enumerate((8, 29, 30)):
        rk, rv = read_rows(kv, b, r + 1)
        close(rk[r], ek[b], 2e-6)
        assert np.array_equal(rv[r], v[b].astype(np.float64))
    kv.ctx.check_device_error()


@pytest.mark.parametrize("dtype,heads,window", [("bf16", 64, 100), ("f16", 64, 17), ("bf16", 32, 1)])
def test_attend_windows_with_a_share_per_team(dtype, heads, window):
    """More segments than SMs, a window that begins inside a tile; with 16 heads two warps share each."""
    lens = [int(n) for n in np.random.default_rng(53).integers(0, 400, 50)]
    test_attend(lens, heads, 4, 128, 16, dtype, window)
    test_attend_accumulates_the_weights(lens, heads, 4, 128, 16, dtype, window)


@pytest.mark.parametrize("dtype,hd,page,gap", [("f16", 128, 16, 8), ("bf16", 64, 64, 4096), ("f32", 64, 16, 4)])
def test_pages_further_apart_than_their_size(dtype, hd, page, gap):
    rng = np.random.default_rng(54)
    lens = [70, 5, 0, 33]
    kv, ks, vs = make_cache(rng, lens, 2, hd, page, dtype, gap=gap)
    assert kv.k.stride(0) == 2 * page * hd + gap
    q = queries(rng, 4, 8, hd)
    close(kv.attend(T(q)).cpu().numpy(), attend_ref(q, ks, vs, hd ** -0.5)[0], 1e-5)
    acc = rng.exponential(1, (4, 2, kv.max_rows)).astype(np.float32)
    pos = np.broadcast_to(np.arange(kv.max_rows, dtype=np.int32), acc.shape)
    _, _, n = kv.evict(T(acc), T(pos), T(np.array(lens, np.int32)), 20, 4, 2)
    assert n.tolist() == [20, 5, 0, 20]
    for b, m in enumerate(lens):
        if m:
            gk, gv = read_rows(kv, b, min(m, 20))
            for j in range(2):
                src = evict_ref(acc[b, j], pos[b, j], m, m, 20, 4, 2)
                assert np.array_equal(gk[:, j], ks[b][src, j]) and np.array_equal(gv[:, j], vs[b][src, j])
    kv.lens = n
    x = T(rng.normal(0, 1, (4, 2, hd)).astype(np.float32))
    kv.append(None, x, x, torch.zeros(4, dtype=torch.int32, device=DEV), 1e4)
    for b, m in enumerate(n.tolist()):
        if m:
            assert np.array_equal(read_rows(kv, b, m)[1][m - 1], x[b].to(TYPES[dtype]).double().cpu().numpy())
    kv.ctx.check_device_error()


def test_sample_refuses_outputs_over_its_inputs():
    """All rows' settings are read to order the rows; u may be overwritten in place."""
    n, v = 40, 500
    rng = np.random.default_rng(55)
    x, u = T(rng.normal(0, 2, (n, v)).astype(np.float32)), T(rng.uniform(0, 1, n).astype(np.float32))
    one = lambda value: torch.full((n,), value, device=DEV)                     # noqa: E731
    t, p, m, k = one(0.9), one(0.8), one(0.01), torch.full((n,), 30, dtype=torch.int32, device=DEV)
    both = torch.zeros(2 * n, device=DEV)
    i = lambda a: a.view(torch.int32)                                           # noqa: E731
    for kw in (dict(token=k), dict(logprob=t), dict(logprob=p), dict(logprob=m), dict(token=i(t)), dict(logprob=k.view(torch.float32)),
               dict(logprob=x.view(-1)[v * n - n:]), dict(token=i(x).view(-1)[:n]),
               dict(token=i(both)[:n], logprob=both[n - 1:2 * n - 1])):
        with pytest.raises(StyxError, match="overlaps") as e:
            ops.sample(x, u, t, k, p, m, **kw)
        assert e.value.code == _lib.STYX_EINVAL
    shifted = both[:n]
    shifted.copy_(u)
    with pytest.raises(StyxError, match="overlaps"):
        ops.sample(x, shifted, t, k, p, m, logprob=both[1:n + 1])
    exp = ops.sample(x, u, t, k, p, m)
    got = ops.sample(x, shifted, t, k, p, m, logprob=shifted)
    assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
    ops.ctx(0).check_device_error()


def test_outputs_over_lengths_or_table_are_refused():
    rng = np.random.default_rng(56)
    kv, _, _ = make_cache(rng, [20, 30], 2, 64, 16, "f16")
    room = torch.zeros(8192, dtype=torch.int32, device=DEV)
    lens, table = room[512:514], room[1024:1024 + kv.table.numel()].view(kv.table.shape)
    lens.copy_(kv.lens)
    table.copy_(kv.table)
    over = ops.PagedKV(kv.k, kv.v, table, lens)
    f = lambda at, *shape: room[at:at + int(np.prod(shape))].view(shape).view(torch.float32)   # noqa: E731
    i = lambda at, *shape: room[at:at + int(np.prod(shape))].view(shape)                       # noqa: E731
    q = T(queries(rng, 2, 8, 64))
    acc, pos, nxt = torch.rand(2, 2, 32, device=DEV), torch.zeros(2, 2, 32, dtype=torch.int32, device=DEV), T(np.array([40, 40], np.int32))
    for call in (lambda: over.attend(q, out=f(0, 2, 8, 64)), lambda: over.attend(q, out=f(1024, 2, 8, 64)),
                 lambda: over.attend(q, lse=f(500, 2, 8)), lambda: over.attend(q, acc=acc, acc_out=f(400, 2, 2, 32)),
                 lambda: over.attend(q, acc=acc, acc_out=f(1020, 2, 2, 32)),
                 lambda: over.evict(acc, pos, nxt, 8, acc_out=f(1020, 2, 2, 32)), lambda: over.evict(acc, pos, nxt, 8, pos_out=i(1020, 2, 2, 32)),
                 lambda: over.evict(acc, pos, nxt, 8, lens_out=i(1024, 2))):
        with pytest.raises(StyxError, match="lens or the table") as e:
            call()
        assert e.value.code == _lib.STYX_EINVAL
    with pytest.raises(StyxError, match="other arrays"):
        over.evict(acc, pos, nxt, 8, acc_out=f(400, 2, 2, 32))
    assert torch.equal(over.attend(q, out=f(4096, 2, 8, 64)), kv.attend(q))
    kv.ctx.check_device_error()
