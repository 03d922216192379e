"""Prompts in chunks over a paged KV cache on the GPU (styx_paged_plan,
styx_paged_append_rope, styx_paged_attend_chunk) against the operators'
definitions in 64 bits (tests/chunk_case.py).

Tolerances, from the arithmetic.  Attention with f32 q: 1e-5 of max|out|, as
for single tokens (scores of size ~10 rounded to f32 move a weight by ~1e-6,
sums of some thousand rows add as much again).  With q of a 16-bit type every
weight p is rounded once, half a step h = eps / 2 of it, and so is the output:
h (sum p |v| + |out|) and the f32 bound.  lse 1e-5 of max(1, |lse|).  Rotated q
and K 2e-6 of the largest (an RMSNorm, a rounded sine and cosine, a magnitude,
three roundings: 7 x 2^-24 and a margin), and half a step of their type.  Plans
are whole numbers: equal.
"""
import numpy as np
import pytest
import torch

from styx_b200 import StyxError, _lib, ops
from tests.chunk_case import Tables, chunk_ref, freqs_ref, turned_ref
from tests.paged_case import DEV, TYPES, make_cache, read_rows

pytestmark = pytest.mark.gpu


def T(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def I(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def queries(rng, n, h, hd, t):
    q = (rng.normal(0, 1, (n, h, hd)) * rng.uniform(0.3, 3, (1, h, 1))).astype(np.float32)
    return torch.from_numpy(q).to(t).to(DEV)


def starts(news):
    return [0] + np.cumsum(news).tolist()


def check_out(got, lse, q_type, ref, start):
    out, ref_lse, mag = ref
    n = start[-1]
    got, lse = got.double().cpu().numpy()[:n], lse.cpu().numpy()[:n]
    assert np.all(np.isfinite(got))
    h = 0.0 if q_type == "f32" else torch.finfo(TYPES[q_type]).eps / 2
    tol = 1e-5 * np.abs(out[:n]).max(initial=1e-30) + h * (mag[:n] + np.abs(out[:n]) * (1 + h))
    err = np.abs(got - out[:n])
    assert np.all(err <= tol), f"{np.max(err / tol):.2f} of the tolerance"
    assert np.all(np.abs(lse - ref_lse[:n]) <= 1e-5 * np.maximum(1, np.abs(ref_lse[:n])))


# ------------------------------------------------------------------ attention
CASES = [
    # rows, new tokens, heads, kv heads, head_dim, page, cache, q, window
    ([1], [1], 32, 4, 128, 16, "f16", "f32", 0),
    ([37], [5], 32, 4, 128, 16, "f16", "f16", 0),
    ([37], [37], 32, 4, 128, 16, "bf16", "f32", 0),
    ([0, 1, 15, 16, 17, 63, 64, 65], [0, 1, 15, 2, 17, 63, 1, 64], 8, 2, 128, 16, "bf16", "bf16", 0),
    ([300, 3, 0, 129, 128], [129, 3, 0, 1, 128], 16, 2, 128, 64, "f16", "f32", 0),
    ([300, 3, 0, 129, 128], [129, 3, 0, 1, 128], 16, 1, 128, 64, "bf16", "bf16", 0),
    ([300, 3, 0, 129, 128], [129, 3, 0, 1, 128], 8, 2, 128, 64, "f32", "f32", 0),
    ([700, 513], [100, 257], 4, 1, 128, 32, "f16", "f16", 300),
    ([700, 513], [100, 257], 4, 1, 128, 32, "bf16", "f32", 33),
    ([300, 20, 1], [300, 2, 1], 4, 2, 128, 256, "f32", "f32", 17),
    ([200, 66], [90, 66], 4, 4, 64, 16, "f16", "f16", 1),
    ([200, 66], [90, 66], 6, 6, 64, 16, "bf16", "bf16", 0),
    ([257, 90], [257, 11], 14, 2, 80, 16, "bf16", "bf16", 0),
    ([257, 90], [257, 11], 14, 2, 80, 16, "f16", "f32", 0),
    ([130, 61], [41, 61], 5, 1, 96, 32, "f16", "f16", 0),
    ([130, 61], [41, 61], 5, 1, 96, 32, "f32", "f32", 64),
    ([66, 200], [60, 100], 14, 2, 256, 16, "bf16", "bf16", 0),
    ([66, 200], [60, 100], 14, 2, 256, 16, "bf16", "f32", 0),
    ([66, 200], [60, 100], 2, 2, 256, 16, "f16", "f32", 50),
    ([66, 200], [60, 100], 7, 1, 256, 16, "f32", "f32", 0),
    ([70], [70], 40, 1, 120, 64, "f16", "f16", 0),
    ([70, 90], [3, 40], 33, 1, 8, 64, "bf16", "bf16", 0),
    ([50], [20], 200, 1, 40, 64, "bf16", "f32", 0),
    ([50], [20], 300, 1, 16, 64, "f16", "f16", 0),
    ([50], [50], 4, 4, 4, 1, "f32", "f32", 0),
    ([45, 99], [45, 30], 8, 4, 128, 1, "f16", "f16", 50),
    ([45, 99], [45, 30], 8, 4, 64, 2, "bf16", "f32", 0),
    ([600], [70], 2, 1, 64, 4096, "f16", "f16", 0),
    ([4100], [3], 8, 1, 128, 128, "bf16", "bf16", 0),
    ([4100], [3], 8, 1, 128, 128, "f16", "f32", 0),
    ([4100, 1, 2050], [2, 1, 9], 4, 1, 128, 64, "f32", "f32", 0),
    ([2500, 900], [20, 700], 2, 1, 128, 64, "f16", "f16", 1000),
    ([600, 600, 512], [40, 9, 40], 8, 2, 128, 64, "f16", "f32", 0),
    ([150, 40], [12, 5], 200, 1, 64, 64, "f16", "f16", 0),
    ([150, 40], [9, 5], 274, 2, 72, 16, "bf16", "bf16", 60),
    ([600, 600, 512], [40, 9, 40], 8, 2, 128, 64, "bf16", "bf16", 400),
    ([1300], [4], 2, 1, 256, 16, "bf16", "bf16", 0),         # (forty portions and more of one segment)
    ([1300], [3], 3, 1, 192, 32, "f32", "f32", 0),
]


@pytest.mark.parametrize("lens,news,heads,n_kv,hd,page,dtype,q_type,window", CASES)
def test_attend_chunk(lens, news, heads, n_kv, hd, page, dtype, q_type, window):
    rng = np.random.default_rng(sum(lens) + heads + hd)
    kv, ks, vs = make_cache(rng, lens, n_kv, hd, page, dtype)
    start = starts(news)
    n = start[-1] + 3                       # three tokens behind the last sequence's
    q = queries(rng, n, heads, hd, TYPES[q_type])
    ref = chunk_ref(q.double().cpu().numpy(), start, ks, vs, hd ** -0.5, window)
    out = torch.full((n, heads, hd), 7.0, device=DEV, dtype=TYPES[q_type])
    lse = torch.full((n, heads), 7.0, device=DEV)
    assert kv.attend_chunk(q, I(start), window=window, out=out, lse=lse) is out
    kv.ctx.check_device_error()
    check_out(out, lse, q_type, ref, start)
    assert torch.all(out[start[-1]:] == 7) and torch.all(lse[start[-1]:] == 7)
    again = kv.attend_chunk(q, I(start), window=window)
    assert torch.equal(again[:start[-1]], out[:start[-1]])          # the same bits, call after call


@pytest.mark.parametrize("dtype,q_type", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
def test_one_token_per_sequence_is_what_attend_does(dtype, q_type):
    rng = np.random.default_rng(1)
    lens = [0, 1, 64, 300, 129, 1000]
    kv, _, _ = make_cache(rng, lens, 4, 128, 64, dtype)
    q = queries(rng, 6, 32, 128, TYPES[q_type])
    one = kv.attend(q.float())
    got = kv.attend_chunk(q[1:].contiguous(), I([0, 0, 1, 2, 3, 4, 5])).float()
    h = 0.0 if q_type == "f32" else torch.finfo(TYPES[q_type]).eps
    assert (got - one[1:]).abs().max() <= (2e-5 + 3 * h) * one.abs().max()
    kv.ctx.check_device_error()


@pytest.mark.parametrize("dtype,q_type", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32"), ("f32", "f32")])
def test_what_a_token_does_not_see_is_not_used(dtype, q_type):
    """NaN and infinities in rows of later tokens, in rows before the window
    and past the end: the tokens that do not see them are untouched; those that
    do have them in their outputs."""
    rng = np.random.default_rng(2)
    lens, news, hd, window = [200, 150], [120, 150], 64, 90
    kv, ks, vs = make_cache(rng, lens, 2, hd, 16, dtype)
    start = starts(news)
    q = queries(rng, start[-1], 8, hd, TYPES[q_type])
    for b, row, bad_k, bad_v in ((0, 150, None, float("nan")), (0, 30, float("nan"), float("inf")), (1, 100, None, float("-inf")),
                                 (1, 149, float("nan"), None)):
        p, at = int(kv.table[b, row // 16]), row % 16
        if bad_v is not None:
            kv.v[p, :, at, 5] = bad_v
            vs[b][row, :, 5] = bad_v
        if bad_k is not None:
            kv.k[p, :, at] = bad_k
            ks[b][row] = bad_k
    lse = torch.zeros(start[-1], 8, device=DEV)
    got = kv.attend_chunk(q, I(start), window=window, lse=lse).double().cpu().numpy()
    kv.ctx.check_device_error()
    with np.errstate(all="ignore"):
        out, ref_lse, mag = chunk_ref(q.double().cpu().numpy(), start, ks, vs, hd ** -0.5, window)
    fine = np.isfinite(out)
    assert not fine.all() and fine.any()
    assert np.all(np.isfinite(got[fine])) and not np.any(np.isfinite(got[~fine]))
    h = 0.0 if q_type == "f32" else torch.finfo(TYPES[q_type]).eps / 2
    tol = 1e-5 * np.abs(out[fine]).max() + h * (mag[fine] + np.abs(out[fine]) * (1 + h))
    assert np.all(np.abs(got[fine] - out[fine]) <= tol)
    ok = np.isfinite(ref_lse)
    got_lse = lse.cpu().numpy()
    assert np.array_equal(np.isfinite(got_lse), ok) and np.all(np.abs(got_lse[ok] - ref_lse[ok]) <= 1e-4)


@pytest.mark.parametrize("dtype,q_type", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32"), ("f32", "f32")])
def test_sharp_and_flat_heads(dtype, q_type):
    """One row with all the weight (scores of +-200: every other weight
    underflows), and equal rows (the mean of V)."""
    rng = np.random.default_rng(4)
    kv, ks, vs = make_cache(rng, [333], 2, 128, 32, dtype)
    q = np.zeros((40, 16, 128), np.float32)
    for t in range(40):
        for h in range(8):
            q[t, h] = ks[0][40 * h, 0] * (20.0 if t % 2 else -20.0)
    q = torch.from_numpy(q).to(TYPES[q_type]).to(DEV)
    ref = chunk_ref(q.double().cpu().numpy(), [0, 40], ks, vs, 128 ** -0.5)
    got = kv.attend_chunk(q, I([0, 40])).double().cpu().numpy()
    h = 0.0 if q_type == "f32" else torch.finfo(TYPES[q_type]).eps / 2
    # scores up to 230 in f32: 2^-24 x 230 x 4 of a weight
    assert np.all(np.abs(got - ref[0]) <= 6e-5 * np.abs(ref[0]).max() + h * (ref[2] + np.abs(ref[0]) * (1 + h)))


@pytest.mark.parametrize("dtype,q_type", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("rise", [0.0, 30.0, 200.0, -200.0])
def test_long_portions_and_rising_scores(dtype, q_type, rise):
    """Enough tiles that every worker has many of one segment in a row, and
    scores that rise (or fall) by `rise` from the first row to the last: what a
    row is measured against has to move, in tiles of every kind."""
    rng = np.random.default_rng(12)
    lens, news, heads, n_kv, hd, page = [2050, 1100, 2304, 700], [300, 290, 310, 700], 16, 8, 128, 64
    kv, ks, vs = make_cache(rng, lens, n_kv, hd, page, dtype)
    start = starts(news)
    q = torch.from_numpy(rng.normal(0, 1, (start[-1], heads, hd)).astype(np.float32))
    q[..., 0] = 8.0
    q = q.to(TYPES[q_type]).to(DEV)
    for b, n in enumerate(lens):      # score += 8 K[r][0] / sqrt(128)
        step = torch.arange(n, dtype=torch.float64) * (rise * 128 ** 0.5 / 8 / max(lens))
        k0 = step.to(torch.float32).to(TYPES[dtype])
        r = torch.arange(n)
        kv.k[kv.table[b].long().cpu()[r // page].to(DEV), :, (r % page).to(DEV), 0] = k0.to(DEV)[:, None]
        ks[b][:, :, 0] = k0.double().numpy()[:, None]
    lse = torch.zeros(start[-1], heads, device=DEV)
    got = kv.attend_chunk(q, I(start), lse=lse).double()
    kv.ctx.check_device_error()
    h = 0.0 if q_type == "f32" else torch.finfo(TYPES[q_type]).eps / 2
    f32 = 1e-5 + 2.0 ** -24 * 4 * abs(rise)          # scores of that size in f32: 2^-24 x 4 of them move a weight
    for b, n in enumerate(lens):
        k, v = T(ks[b]), T(vs[b])
        at = slice(start[b], start[b + 1])
        x = torch.einsum("tjgd,rjd->jgtr", q[at].double().unflatten(1, (n_kv, 2)), k) * hd ** -0.5
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - news[b], n, device=DEV)[:, None]
        x.masked_fill_(hidden, -torch.inf)
        p = torch.softmax(x, -1)
        out = torch.einsum("jgtr,rjd->tjgd", p, v).flatten(1, 2)
        mag = torch.einsum("jgtr,rjd->tjgd", p, v.abs()).flatten(1, 2)
        tol = f32 * out.abs().max() + h * (mag + out.abs() * (1 + h))
        assert ((got[at] - out).abs() <= tol).all(), f"{((got[at] - out).abs() / tol).max().item():.2f} of the tolerance"
        ref = torch.logsumexp(x, -1).permute(2, 0, 1).flatten(1, 2)
        assert ((lse[at].double() - ref).abs() <= 1e-5 * ref.abs().clamp(min=1)).all()
    again = kv.attend_chunk(q, I(start))
    assert torch.equal(again.double(), got)


def test_strided_queries_scales_and_many_segments():
    """q as a slice of a projection's output; another scale; more segments than SMs."""
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(1, 260, 60)]
    news = [int(rng.integers(0, n + 1)) for n in lens]
    for dtype, q_type in (("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")):
        kv, ks, vs = make_cache(rng, lens, 4, 64, 32, dtype)
        start = starts(news)
        wide = queries(rng, start[-1], 24, 64, TYPES[q_type])
        q = wide[:, 4:20]
        assert not q.is_contiguous()
        lse = torch.zeros(start[-1], 16, device=DEV)
        got = kv.attend_chunk(q, I(start), scale=0.3, lse=lse)
        kv.ctx.check_device_error()
        check_out(got, lse, q_type, chunk_ref(q.double().cpu().numpy(), start, ks, vs, 0.3), start)


@pytest.mark.parametrize("dtype,q_type", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
def test_pages_outside_the_pool_and_bad_ranges_are_skipped_and_reported(dtype, q_type):
    rng = np.random.default_rng(6)
    lens, news = [100, 64, 40], [60, 64, 40]
    kv, ks, vs = make_cache(rng, lens, 2, 64, 16, dtype, max_rows=200)
    start = starts(news)
    q = queries(rng, start[-1], 8, 64, TYPES[q_type])
    kv.table[0, 7:] = -7                      # past the end: not looked at
    kv.table[1, 4:] = 1 << 30
    good = kv.attend_chunk(q, I(start))
    kv.ctx.check_device_error()
    kv.table[0, 2] = kv.k.shape[0]            # rows 32 to 47 of the first
    got = kv.attend_chunk(q, I(start))
    with pytest.raises(StyxError):
        kv.ctx.check_device_error()
    keep = [r for r in range(100) if not 32 <= r < 48]
    k0, v0 = ks[0].copy(), vs[0].copy()
    for t in range(60):
        r = 40 + t
        rows = [x for x in keep if x <= r]
        s = np.einsum("rjd,jgd->jgr", k0[rows], q[t].double().cpu().numpy().reshape(2, 4, 64)) / 8
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        exp = np.einsum("jgr,rjd->jgd", p, v0[rows]).reshape(8, 64)
        h = 0.0 if q_type == "f32" else torch.finfo(TYPES[q_type]).eps
        assert np.abs(got[t].double().cpu().numpy() - exp).max() <= (2e-5 + 2 * h) * np.abs(v0).max()
    assert torch.equal(got[60:], good[60:])
    # ranges that are none: those sequences are left out, the others done
    for bad in ([0, 101, 164, 164], [0, 60, 50, 164], [0, 60, 124, 165], [-1, 60, 124, 164]):
        out = torch.full_like(q, 7.0)
        kv.table[0, 2] = 0
        kv.attend_chunk(q, I(bad), out=out)
        with pytest.raises(StyxError):
            kv.ctx.check_device_error()
        kv.ctx.check_device_error()


def test_chunk_refusals():
    rng = np.random.default_rng(7)
    kv, _, _ = make_cache(rng, [10, 20], 2, 64, 16, "f16")
    q, start = queries(rng, 8, 8, 64, torch.float16), I([0, 4, 8])
    with pytest.raises(ValueError):
        kv.attend_chunk(q.bfloat16(), start)
    with pytest.raises(ValueError):
        kv.attend_chunk(q, I([0, 8]))
    with pytest.raises(ValueError):
        kv.attend_chunk(q, start, out=torch.zeros(8, 8, 64, device=DEV))
    with pytest.raises(ValueError):
        kv.attend_chunk(q.cpu(), start)
    with pytest.raises(ValueError):
        kv.attend_chunk(q[..., ::2], start)
    with pytest.raises(StyxError):
        kv.attend_chunk(q[:, :7], start)                        # 7 heads over 2
    with pytest.raises(StyxError):
        kv.attend_chunk(q, start, out=q)
    with pytest.raises(StyxError):
        kv.attend_chunk(q, start, window=-1)
    with pytest.raises(StyxError):
        kv.attend_chunk(q, start, scale=float("inf"))
    flat = torch.zeros(8 * 8 * 64 + 8, device=DEV, dtype=torch.float16)
    with pytest.raises(StyxError):                              # tokens 16-byte aligned only at the first
        kv.attend_chunk(torch.as_strided(flat, (7, 8, 64), (516, 64, 1)), start)
    with pytest.raises(StyxError):
        kv.attend_chunk(flat[1:1 + 8 * 512].view(8, 8, 64), start)
    n = kv._attend_ws
    kv.attend_chunk(q, start)
    (t, at, nb), = [v for k, v in n.items() if k[-1] == "chunk"]
    L, out = kv._lib, torch.empty_like(q)
    args = (kv.ctx.handle, None, kv._ref, 8, 8, _lib.F16, q.data_ptr(), 512, start.data_ptr(), 0.125, 0)
    assert L.styx_paged_attend_chunk(*args, out.data_ptr(), None, at, nb - 256) == _lib.STYX_EINVAL
    assert L.styx_paged_attend_chunk(*args, out.data_ptr(), None, at + 16, nb) == _lib.STYX_EINVAL
    assert L.styx_paged_attend_chunk(*args, out.data_ptr(), out.data_ptr(), at, nb) == _lib.STYX_EINVAL
    assert L.styx_paged_attend_chunk(*args, kv.table.data_ptr(), None, at, nb) == _lib.STYX_EINVAL
    assert L.styx_paged_attend_chunk(*args, out.data_ptr(), None, at, nb) == 0
    torch.cuda.synchronize()


def test_chunk_on_another_stream_and_in_a_graph():
    """A captured call follows the lengths, the ranges and the rows that its replays find."""
    rng = np.random.default_rng(8)
    for dtype, q_type in (("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")):
        kv, ks, vs = make_cache(rng, [150, 90], 2, 64, 16, dtype)
        lens = kv.lens.clone()
        start = I([0, 50, 100])
        q = queries(rng, 100, 8, 64, TYPES[q_type])
        out, lse = torch.zeros_like(q), torch.zeros(100, 8, device=DEV)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        kv.attend_chunk(q, start, out=out, lse=lse, stream=s)
        s.synchronize()
        first = out.clone()
        check_out(out, lse, q_type, chunk_ref(q.double().cpu().numpy(), [0, 50, 100], ks, vs, 0.125), [0, 50, 100])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv.attend_chunk(q, start, out=out, lse=lse)
        for n0, n1, at in ((150, 90, [0, 50, 100]), (60, 90, [0, 60, 61]), (1, 0, [0, 1, 1]), (149, 33, [0, 0, 33])):
            kv.lens.copy_(I([n0, n1]))
            start.copy_(I(at))
            out.zero_()
            lse.zero_()
            g.replay()
            ref = chunk_ref(q.double().cpu().numpy(), at, [ks[0][:n0], ks[1][:n1]], [vs[0][:n0], vs[1][:n1]], 0.125)
            check_out(out, lse, q_type, ref, at)
            assert not out[at[-1]:].any()
        kv.lens.copy_(lens)
        start.copy_(I([0, 50, 100]))
        g.replay()
        assert torch.equal(out, first)
        kv.ctx.check_device_error()


def test_many_calls_of_ragged_batches():
    """Calls back to back, lengths and ranges of one after the other: each
    gives the bits that it gives alone, and no wait gives up."""
    rng = np.random.default_rng(13)
    for dtype, q_type, hd in (("bf16", "bf16", 128), ("f16", "f32", 128), ("f16", "f16", 64)):
        kv, _, _ = make_cache(rng, [1500] * 24, 4, hd, 64, dtype)
        n = 700
        q = queries(rng, n, 32, hd, TYPES[q_type])
        sets = []
        for _ in range(6):
            lens = np.where(rng.random(24) < 0.2, 0, rng.integers(1, 1501, 24))
            news = np.minimum(lens, np.where(rng.random(24) < 0.5, rng.integers(1, 8, 24), rng.integers(1, 50, 24)))
            news[np.cumsum(news) > n] = 0
            sets.append((I(lens.tolist()), I(starts(news.tolist()))))
        alone = []
        for lens, start in sets:
            kv.lens = lens
            alone.append(kv.attend_chunk(q, start, out=torch.zeros_like(q)))
            torch.cuda.synchronize()
        outs = [torch.zeros_like(q) for _ in sets]
        for i in range(600):
            kv.lens = sets[i % 6][0]
            kv.attend_chunk(q, sets[i % 6][1], out=outs[i % 6])
        kv.ctx.check_device_error()
        for a, b in zip(alone, outs):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ append with rotary forms
@pytest.mark.parametrize("hd,n_dims", [(128, 128), (128, 64), (128, 112), (64, 64), (80, 40), (80, 20), (96, 96), (256, 64),
                                       (8, 8), (8, 2), (40, 18), (4, 4)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype,q_type", [("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
def test_append_rope(hd, n_dims, inter, dtype, q_type):
    if hd == 4 and dtype != "f32":
        pytest.skip("16-bit rows of 8 bytes")
    rng = np.random.default_rng(hd + n_dims)
    heads, n_kv, page, n = 6, 2, 16, 37
    kv, _, _ = make_cache(rng, [60, 0, 40], n_kv, hd, page, dtype)
    seq = np.array([0] * 20 + [2] * 17, np.int32)
    row = np.concatenate([np.arange(40, 60), np.arange(23, 40)]).astype(np.int32)
    row[5] = -1
    pos = rng.integers(0, 200000, n).astype(np.int32)
    qkv = rng.normal(0, 1, (n, (heads + 2 * n_kv) * hd)).astype(np.float32)
    q, k, v = (t.unflatten(1, (-1, hd)) for t in T(qkv).split([heads * hd, n_kv * hd, n_kv * hd], 1))
    qw, kw = rng.uniform(0.5, 1.5, (2, hd)).astype(np.float32)
    factors = rng.uniform(1, 8, n_dims // 2).astype(np.float32)
    rope = ops.Rope(n_dims, 1e6, inter, "yarn", 4.0, 32768, factors=torch.from_numpy(factors))
    freq, grow = freqs_ref(n_dims, 1e6, "yarn", 4.0, 32768, factors=factors)
    before = [read_rows(kv, b, m) for b, m in ((0, 60), (2, 40))]
    out = torch.empty(n, heads, hd, device=DEV, dtype=TYPES[q_type])
    assert kv.append(q, k, v, T(pos), rope=rope, q_norm=T(qw), k_norm=T(kw), eps=1e-6, seq=T(seq), row=T(row), out=out) is out
    kv.ctx.check_device_error()
    f64 = [t.double().cpu().numpy() for t in (q, k, v)]
    rq = turned_ref(f64[0], qw, pos, freq, n_dims, inter, grow, 1e-6)
    rk = turned_ref(f64[1], kw, pos, freq, n_dims, inter, grow, 1e-6)
    rq[5] = 0
    half = {t: 0.0 if t == "f32" else torch.finfo(TYPES[t]).eps / 2 for t in TYPES}
    err = np.abs(out.double().cpu().numpy() - rq)
    # (f16: half a step of the smallest numbers too)
    tiny = {t: 2.0 ** -25 if t == "f16" else 0.0 for t in TYPES}
    assert np.all(err <= 2e-6 * np.abs(rq).max() * (1 + half[q_type]) + half[q_type] * np.abs(rq) + tiny[q_type])
    for (b, m), was in zip(((0, 60), (2, 40)), before):
        gk, gv = read_rows(kv, b, m)
        ek, ev = was
        written = np.zeros(m, bool)
        for t in range(n):
            if seq[t] == b and row[t] >= 0:
                ek[row[t]], ev[row[t]] = rk[t], f64[2][t]
                written[row[t]] = True
        assert np.array_equal(gk[~written], ek[~written]) and np.array_equal(gv[~written], ev[~written])
        h = half[dtype]
        assert np.all(np.abs(gk - ek)[written] <= 2e-6 * np.abs(rk).max() * (1 + h) + h * np.abs(ek[written]) + tiny[dtype])
        assert np.all(np.abs(gv - ev)[written] <= h * np.abs(ev[written]) + tiny[dtype])


def test_append_rope_over_the_whole_head_is_append():
    rng = np.random.default_rng(9)
    a, _, _ = make_cache(rng, [64, 30], 2, 128, 16, "f16")
    b, _, _ = make_cache(np.random.default_rng(9), [64, 30], 2, 128, 16, "f16")
    q, k, v = (T(rng.normal(0, 1, (2, h, 128)).astype(np.float32)) for h in (8, 2, 2))
    pos, w = I([63, 70000]), T(rng.uniform(0.5, 1.5, 128).astype(np.float32))
    one = a.append(q, k, v, pos, 1e6, w, w)
    two = b.append(q, k, v, pos, rope=ops.Rope(128, 1e6), q_norm=w, k_norm=w)
    # the same formula from frequencies that differ by a few units of 2^-53
    assert (one - two).abs().max() <= 2.0 ** -22 * one.abs().max()
    same = (a.k.view(torch.int16) - b.k.view(torch.int16)).abs()
    assert same.max() <= 1 and torch.equal(a.v.view(torch.int16), b.v.view(torch.int16))


def test_append_rope_passes_what_it_does_not_turn():
    """Elements behind n_dims, and all of V, come out as they went in, whatever their neighbours hold."""
    kv, _, _ = make_cache(np.random.default_rng(0), [3], 1, 64, 16, "f32")
    for inter in (False, True):
        x = torch.randn(1, 1, 64, device=DEV)
        x[0, 0, 33], x[0, 0, 40] = float("nan"), float("inf")
        got = kv.append(x, x, x, I([5]), rope=ops.Rope(32, 1e4, inter))
        keep = torch.tensor([i for i in range(32, 64)], device=DEV)
        row = kv.k[int(kv.table[0, 0]), 0, 2]
        for y in (got[0, 0], row):
            assert torch.equal(y[keep].view(torch.int32), x[0, 0, keep].view(torch.int32)) and y[:32].isfinite().all()
        assert torch.equal(kv.v[int(kv.table[0, 0]), 0, 2].view(torch.int32), x[0, 0].view(torch.int32))


def test_append_rope_refusals():
    kv, _, _ = make_cache(np.random.default_rng(0), [3, 3], 2, 64, 16, "f16")
    q, k, pos = torch.zeros(2, 8, 64, device=DEV), torch.zeros(2, 2, 64, device=DEV), I([0, 0])
    rope = ops.Rope(64, 1e4)
    with pytest.raises(ValueError):
        kv.append(q, k, k, pos)
    with pytest.raises(ValueError):
        kv.append(q, k, k, pos, 1e4, rope=rope)
    with pytest.raises(ValueError):
        kv.append(q, k, k, pos, 1e4, out=torch.zeros(2, 8, 64, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        kv.append(q, k, k, pos, rope=rope, out=torch.zeros(2, 8, 64, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(StyxError):
        kv.append(q, k, k, pos, rope=ops.Rope(66, 1e4))
    with pytest.raises(StyxError):
        kv.append(q, k, k, pos, rope=rope, out=q)
    for field, value in (("n_dims", 63), ("n_dims", 0), ("freq", None)):
        r = ops.Rope(64, 1e4)
        setattr(r._form, field, value)
        with pytest.raises(StyxError):
            kv.append(q, k, k, pos, rope=r)
    kv.append(q, k, k, pos, rope=rope)
    kv.append(q, k, k, I([0, 0]), rope=rope, row=I([3, 1 << 20]))
    with pytest.raises(StyxError):
        kv.ctx.check_device_error()


# ------------------------------------------------------------------ plans
def plan_of(t, n_tokens):
    table, free = T(t.table), T(t.free)
    return ops.PagedPlan(table, t.page, free, n_tokens)


def same(p, t, got, n_tokens):
    start, seq, row, pos = got
    assert p.start.tolist() == start.tolist()
    for a, b in ((p.seq, seq), (p.row, row), (p.pos, pos)):
        assert np.array_equal(a.cpu().numpy(), b)
    assert p.lens.tolist() == t.lens and p.held.tolist() == t.held and p.n_free.item() == t.n_free
    assert p.next_pos.tolist() == t.next_pos
    assert np.array_equal(p.table.cpu().numpy(), t.table)
    assert np.array_equal(p.free.cpu().numpy(), t.free)


@pytest.mark.parametrize("n,max_pages,page,n_tokens,spare", [
    (1, 4, 16, 7, 4), (1, 1, 1, 3, 0), (3, 5, 16, 20, 3), (64, 32, 16, 64, 10), (64, 32, 16, 4096, 100), (64, 32, 16, 4097, 5),
    (200, 64, 4, 9000, 400), (1024, 8, 8, 2000, 300), (1025, 8, 8, 2000, 300), (2500, 6, 4, 5000, 50), (33, 4, 4096, 30000, 20),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(n, max_pages, page, n_tokens, spare, in_place):
    rng = np.random.default_rng(n + n_tokens)
    most = max_pages * page
    lens = np.minimum(most, np.floor(np.exp(rng.uniform(0, np.log(most + 1), n))).astype(int) - 1 + rng.integers(0, 2, n))
    held = np.minimum(max_pages, -(-lens // page) + rng.integers(0, 2, n))
    t = Tables(rng, n, max_pages, page, int(held.sum()) + spare, lens, held)
    p = plan_of(t, n_tokens)
    lens, held, n_free, nxt = I(t.lens), I(t.held), I([t.n_free]), I(t.next_pos)
    if in_place:
        for dst, src in ((p.lens, lens), (p.held, held), (p.n_free, n_free), (p.next_pos, nxt)):
            dst.copy_(src)
    for step in range(4):
        want = rng.choice([-3, 0, 1, 1, 2, page, most, 2 ** 31 - 1], n)
        if step == 2:
            done = rng.random(n) < 0.4                     # finished: their pages go back
            want[done] = 0
            for b in np.nonzero(done)[0]:
                t.lens[b] = 0
        if in_place:
            p.lens.copy_(I(t.lens))
            p.run(I(want.tolist()), p.lens, p.held, p.n_free, p.next_pos)
            same(p, t, t.plan(want, n_tokens), n_tokens)
        else:
            lens = I(t.lens)
            p.run(I(want.tolist()), lens, held, n_free, nxt)
            got = t.plan(want, n_tokens)
            same(p, t, got, n_tokens)
            assert p.run(I(want.tolist()), lens, held, n_free, nxt) is p     # the same inputs: the same results
            same(p, t, got, n_tokens)
            held, n_free, nxt = p.held.clone(), p.n_free.clone(), p.next_pos.clone()
    p.ctx.check_device_error()
    # no page twice
    used = [i for b in range(n) for i in t.table[b, :t.held[b]].tolist()] + t.free[:t.n_free].tolist()
    assert sorted(used) == list(range(len(t.free)))


def test_plan_without_positions_and_in_a_graph():
    rng = np.random.default_rng(3)
    t = Tables(rng, 5, 6, 8, 20, [0, 3, 8, 0, 17], [0, 1, 1, 0, 3])
    p = plan_of(t, 40)
    p.lens.copy_(I(t.lens))
    p.held.copy_(I(t.held))
    p.n_free.copy_(I([t.n_free]))
    want = I([0] * 5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    p.run(want, p.lens, p.held, p.n_free, stream=s)
    s.synchronize()
    t.plan([0] * 5, 40)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.run(want, p.lens, p.held, p.n_free)
    for w in ([1, 1, 1, 1, 1], [30, 2, 0, 5, 9], [0, 40, 40, 1, 1]):
        want.copy_(I(w))
        g.replay()
        t.next_pos = list(t.lens)
        start, seq, row, _ = t.plan(w, 40)
        assert p.start.tolist() == start.tolist() and p.row.tolist() == row.tolist() and p.seq.tolist() == seq.tolist()
        assert p.pos.tolist() == [max(r, 0) for r in row.tolist()]
        assert p.lens.tolist() == t.lens and p.held.tolist() == t.held and p.n_free.item() == t.n_free
    p.ctx.check_device_error()


def test_plan_reports_what_contradicts_itself():
    table, free = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4).contiguous(), torch.full((20,), -1, dtype=torch.int32, device=DEV)
    free[:4] = I([12, 13, 14, 15])
    p = ops.PagedPlan(table, 4, free, 16)
    for lens, held, n_free in (([-1, 4, 4], [1, 1, 1], 4), ([5, 4, 4], [1, 1, 1], 4), ([4, 4, 4], [1, 1, 5], 4), ([4, 4, 4], [-1, 1, 1], 4)):
        p.run(I([2, 2, 2]), I(lens), I(held), I([n_free]))
        with pytest.raises(StyxError):
            p.ctx.check_device_error()
        bad = [not (0 <= h <= 4 and 0 <= n <= 4 * h) for n, h in zip(lens, held)]
        assert p.lens.tolist() == [n if x else n + 2 for n, x in zip(lens, bad)]
        assert p.held.tolist() == [h if x else h + 1 for h, x in zip(held, bad)]
    for n_free in (-1, 21):
        p.run(I([0, 0, 0]), I([4, 4, 4]), I([1, 1, 1]), I([n_free]))
        with pytest.raises(StyxError):
            p.ctx.check_device_error()


def test_plan_refusals():
    table, free, one = torch.zeros(3, 4, dtype=torch.int32, device=DEV), torch.zeros(20, dtype=torch.int32, device=DEV), I([0, 0, 0])
    for bad in (0, 3, 8192):
        with pytest.raises(StyxError):
            ops.PagedPlan(table, bad, free, 16).run(one, one, one, I([0]))
    with pytest.raises(ValueError):
        ops.PagedPlan(table.long(), 4, free, 16)
    with pytest.raises(ValueError):
        ops.PagedPlan(table, 4, free.long(), 16)
    with pytest.raises(ValueError):
        ops.PagedPlan(table, 4, free, 0)
    p = ops.PagedPlan(table, 4, free, 16)
    with pytest.raises(ValueError):
        p.run(one[:2], one, one, I([0]))
    with pytest.raises(StyxError):
        p.run(one, p.held, one, I([0]))
    with pytest.raises(StyxError):
        p.run(p.lens, one, one, I([0]))
    with pytest.raises(StyxError):
        p.run(one, one, one, p.free[:1])
    p.run(one, one, one, I([0]))
    p.ctx.check_device_error()


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype,q_type", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
def test_prompts_in_chunks_are_whole_prompts(dtype, q_type):
    """Plan, append and attention, a budget of tokens at a time, give every
    token what the definition gives over the whole prompts."""
    rng = np.random.default_rng(11)
    prompts, hd, page, heads, n_kv, budget = [70, 1, 33, 0, 129], 64, 16, 8, 2, 48
    width = 10
    n_pages = 40
    k = torch.full((n_pages, n_kv, page, hd), float("nan"), dtype=TYPES[dtype], device=DEV)
    v = torch.full_like(k, float("nan"))
    table = torch.full((5, width), -1, dtype=torch.int32, device=DEV)
    free = T(rng.permutation(n_pages).astype(np.int32))
    lens = torch.zeros(5, dtype=torch.int32, device=DEV)
    kv = ops.PagedKV(k, v, table, lens)
    plan = ops.PagedPlan(table, page, free, budget)
    for t in (plan.lens, plan.held, plan.next_pos):
        t.zero_()
    plan.n_free.fill_(n_pages)
    kv.lens = plan.lens
    rope = ops.Rope(32, 1e4, True, "linear", 2.0)
    freq, _ = freqs_ref(32, 1e4, "linear", 2.0)
    xq, xk, xv = ([rng.normal(0, 1, (n, h, hd)).astype(np.float32) for n in prompts] for h in (heads, n_kv, n_kv))
    left, done, outs = list(prompts), [0] * 5, [[] for _ in prompts]
    while any(left):
        plan.run(I(left), plan.lens, plan.held, plan.n_free, plan.next_pos)
        start = plan.start.tolist()
        took = [start[b + 1] - start[b] for b in range(5)]
        rows = [torch.zeros(budget, h, hd, device=DEV) for h in (heads, n_kv, n_kv)]
        for x, src in zip(rows, (xq, xk, xv)):
            for b in range(5):
                x[start[b]:start[b + 1]] = T(src[b][done[b]:done[b] + took[b]])
        q = torch.empty(budget, heads, hd, device=DEV, dtype=TYPES[q_type])
        kv.append(rows[0], rows[1], rows[2], plan.pos, rope=rope, seq=plan.seq, row=plan.row, out=q)
        got = kv.attend_chunk(q, plan.start)
        for b in range(5):
            outs[b].append(got[start[b]:start[b + 1]].double().cpu().numpy())
            done[b] += took[b]
            left[b] -= took[b]
    kv.ctx.check_device_error()
    assert plan.lens.tolist() == prompts == plan.next_pos.tolist()
    for b, n in enumerate(prompts):
        if not n:
            continue
        pos = np.arange(n)
        rq = torch.from_numpy(turned_ref(xq[b].astype(np.float64), None, pos, freq, 32, True, 1.0, 0)).to(TYPES[q_type]).double().numpy()
        ks, vs = read_rows(kv, b, n)
        out, _, mag = chunk_ref(rq, [0, n], [ks], [vs], hd ** -0.5)
        h = 0.0 if q_type == "f32" else torch.finfo(TYPES[q_type]).eps / 2
        # (q may round the other way where the kernel's f32 differs: one step of q moves a score by 2 h |q||k| / 8)
        tol = 1e-5 * np.abs(out).max() + h * (mag + np.abs(out) * (1 + h)) + 2 * h * np.abs(out).max()
        assert np.all(np.abs(np.concatenate(outs[b]) - out) <= tol)
