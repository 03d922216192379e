// paged_rope.cu -- rows into a paged KV cache with any rotary form
// (styx_paged_append_rope): pairs of halves or of neighbours, part of the head,
// frequencies from a table, q in f32 or in the cache's type.
//
// As k_paged_append: a warp takes a token's rows (q heads, k heads, v heads) or
// a share of them, LPR lanes per row, two rows of a lane at a time, all loads
// first.  A lane has four pairs, two runs of four elements each; where the two
// runs are neighbours (pairs of neighbours, and the part of a head that is not
// turned) they are one access of 8 elements.  Which pairs those are does not
// change the norm, which takes the whole row, and is two address computations
// per lane, once.  The angle in turns, pos * freq / 2 pi, is held in 64 bits
// and reduced to a fraction of a turn before it is rounded to f32, so its
// error does not grow with the position.  Bound by HBM on prompts (8191 tokens of
// 32 q and 2 x 4 k / v heads of 128 into bf16 rows, q bf16: 252 MB in 54 us, 4.7
// TB/s), by the latency of position, page and rows on a step of 64 tokens (3.6
// us).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "paged.cuh"

namespace styx {
namespace {

constexpr int kThreads = 128, kRows = 2;

// a lane's four pairs of a row of hd elements, the first n of them turned
struct Lane {
    int at[2];         // its runs of four elements (vectors); else of its pair e: at0(e), at1(e)
    bool apart;        // pair e is (run 0 [e], run 1 [e]); else the pairs are (0, 1), (2, 3) of run 0, then of run 1
    bool in;
};
// pair p of the row: its two elements
__device__ __forceinline__ int2 pair_at(int p, int n, bool inter) {
    if (!inter && p < n / 2) return make_int2(p, p + n / 2);
    return make_int2(2 * p, 2 * p + 1);   // (behind the halves: n + 2 (p - n / 2))
}

template <class T>
__device__ __forceinline__ void put4(T *p, const float (&v)[4]) {
    T u[4] = {from_f<T>(v[0]), from_f<T>(v[1]), from_f<T>(v[2]), from_f<T>(v[3])};
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(u);
    else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(u);
}
template <class T>
__device__ __forceinline__ void put8(T *p, const float (&v)[4], const float (&w)[4]) {
    if constexpr (sizeof(T) == 4) {
        put4(p, v);
        put4(p + 4, w);
    } else {
        T u[8] = {from_f<T>(v[0]), from_f<T>(v[1]), from_f<T>(v[2]), from_f<T>(v[3]),
                  from_f<T>(w[0]), from_f<T>(w[1]), from_f<T>(w[2]), from_f<T>(w[3])};
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(u);
    }
}

// T: the cache's type; TQ: q_out's.  FORM: what all lanes have, halves of the
// whole head or neighbours (known to the compiler: 64 us instead of 54 for the
// prompts above otherwise), both with every run of four elements aligned; SOME
// as the lane's place says; ODD the same by element.  splits: warps per token,
// share rows each.
enum Form { HALVES, NEIGHBOURS, SOME, ODD };
template <class T, class TQ, int LPR, Form FORM>
__global__ void __launch_bounds__(kThreads, 8) k_paged_append_rope(PagedAppendArgs a, PagedRope rope, TQ *q_out, int splits, int share) {
    pdl_trigger();
    constexpr int RPW = 32 / LPR;
    constexpr bool VEC = FORM != ODD;
    const PagedKv &kv = a.kv;
    const int hd = kv.hd, n = rope.n_dims, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int p0 = lane % LPR * 4, sub = lane / LPR, rows = a.n_heads + 2 * kv.n_kv;
    const bool inter = rope.interleaved;
    Lane L;
    L.in = p0 < hd / 2;
    L.apart = FORM == HALVES || (FORM != NEIGHBOURS && !inter && p0 < n / 2);
    L.at[0] = L.apart ? p0 : 2 * p0;
    L.at[1] = L.apart ? p0 + n / 2 : 2 * p0 + 4;
    // the lane's elements, as pairs (x[e], y[e])
    auto get = [&](const float *src, float (&x)[4], float (&y)[4]) {
        if constexpr (VEC) {
            const float4 u = *reinterpret_cast<const float4 *>(src + L.at[0]), v = *reinterpret_cast<const float4 *>(src + L.at[1]);
            x[0] = u.x;
            y[3] = v.w;
            x[1] = L.apart ? u.y : u.z;
            x[2] = L.apart ? u.z : v.x;
            x[3] = L.apart ? u.w : v.z;
            y[0] = L.apart ? v.x : u.y;
            y[1] = L.apart ? v.y : u.w;
            y[2] = L.apart ? v.z : v.y;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (p0 + e < hd / 2) {
                    const int2 i = pair_at(p0 + e, n, inter);
                    x[e] = src[i.x];
                    y[e] = src[i.y];
                }
        }
    };
    pdl_wait();
    // (the frequencies and the norms may be an earlier kernel's)
    const int nt = FORM == HALVES ? 4 : max(0, min(4, n / 2 - p0));   // how many of the lane's pairs are turned
    float wq[2][4], wk[2][4];
#pragma unroll
    for (int e = 0; e < 4; e++) wq[0][e] = wq[1][e] = wk[0][e] = wk[1][e] = 1.f;
    if (L.in) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (p0 + e < hd / 2) {
                const int2 i = pair_at(p0 + e, n, inter);
                if (a.q_norm) wq[0][e] = ld_now(a.q_norm + i.x), wq[1][e] = ld_now(a.q_norm + i.y);
                if (a.k_norm) wk[0][e] = ld_now(a.k_norm + i.x), wk[1][e] = ld_now(a.k_norm + i.y);
            }
    }
    const unsigned units = static_cast<unsigned>(a.n_tokens) * splits;
    for (unsigned u = blockIdx.x * (kThreads / 32) + warp; u < units; u += gridDim.x * (kThreads / 32)) {
        const int t = u / splits, h_begin = (u - t * splits) * share, h_end = min(rows, h_begin + share);
        float x[kRows][4], y[kRows][4];
        auto load = [&](int h0) {
#pragma unroll
            for (int j = 0; j < kRows; j++) {
                const int h = h0 + j * RPW + sub;
#pragma unroll
                for (int e = 0; e < 4; e++) x[j][e] = y[j][e] = 0.f;
                if (h < h_end && L.in) {
                    const int hk = h - a.n_heads;
                    const float *src = hk < 0         ? a.q + t * a.q_stride + static_cast<long long>(h) * hd
                                       : hk < kv.n_kv ? a.k + t * a.k_stride + static_cast<long long>(hk) * hd
                                                      : a.v + t * a.v_stride + static_cast<long long>(hk - kv.n_kv) * hd;
                    get(src, x[j], y[j]);
                }
            }
        };
        load(h_begin);
        const int b = a.seq ? ld_now(a.seq + t) : t, pos = ld_now(a.pos + t);
        const bool seq_ok = static_cast<unsigned>(b) < static_cast<unsigned>(kv.n_seqs);
        const int r = !seq_ok ? -1 : a.row ? ld_now(a.row + t) : ld_now(kv.lens + b) - 1;
        bool row_ok = r >= 0 && r < (static_cast<long long>(kv.max_pages) << kv.page_shift);
        const long long off = row_ok ? paged_off(kv, b, 0, r) : -1;   // of kv head 0
        row_ok = off >= 0;
        if (lane == 0 && h_begin == 0 && (!seq_ok || (r >= 0 && !row_ok))) atomicExch(kv.err, kErrBadPos);
        float c[4], s[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            // (read for every token: in registers all along they cost the occupancy that hides the loads)
            const double f = e < nt && L.in ? pos * (ld_now(rope.freq + p0 + e) * 0.15915494309189535) : 0.0;   // 1 / 2 pi
            sincospif(static_cast<float>(2.0 * (f - rint(f))), &s[e], &c[e]);
            c[e] *= rope.magnitude;
            s[e] *= rope.magnitude;
        }
        for (int h0 = h_begin;;) {
#pragma unroll
            for (int j = 0; j < kRows; j++) {
                const int h = h0 + j * RPW + sub, hk = h - a.n_heads;
                const bool is_q = hk < 0, is_v = hk >= kv.n_kv;
                if (a.q_norm || a.k_norm) {            // (for all lanes: their rows may be of two kinds)
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; e++) ss += x[j][e] * x[j][e] + y[j][e] * y[j][e];
#pragma unroll
                    for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, LPR);
                    const bool normed = is_q ? a.q_norm != nullptr : !is_v && a.k_norm;
                    const float scale = !normed ? 1.f : 1.0f / sqrtf(ss / static_cast<float>(hd) + a.eps);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[j][e] *= scale * (is_v ? 1.f : is_q ? wq[0][e] : wk[0][e]);
                        y[j][e] *= scale * (is_v ? 1.f : is_q ? wq[1][e] : wk[1][e]);
                    }
                }
                float p[4], q[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool as_is = is_v || e >= nt;   // (0 x a NaN of the other element would be one too)
                    p[e] = as_is ? x[j][e] : x[j][e] * c[e] - y[j][e] * s[e];
                    q[e] = as_is ? y[j][e] : x[j][e] * s[e] + y[j][e] * c[e];
                    if (r < 0) p[e] = q[e] = 0.f;          // padding, or an empty slot
                }
                if (h >= h_end || !L.in) continue;
                auto put = [&](auto *o) {
                    if constexpr (VEC) {
                        if (L.apart) {
                            put4(o + L.at[0], p);
                            put4(o + L.at[1], q);
                        } else {
                            const float u[4] = {p[0], q[0], p[1], q[1]}, v[4] = {p[2], q[2], p[3], q[3]};
                            put8(o + L.at[0], u, v);
                        }
                    } else {
                        using O = std::remove_pointer_t<decltype(o)>;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (p0 + e < hd / 2) {
                                const int2 i = pair_at(p0 + e, n, inter);
                                o[i.x] = from_f<O>(p[e]);
                                o[i.y] = from_f<O>(q[e]);
                            }
                    }
                };
                if (is_q) put(q_out + (static_cast<long long>(t) * a.n_heads + h) * hd);
                else if (row_ok)
                    put(static_cast<T *>(is_v ? kv.v : kv.k) + off +
                        (static_cast<long long>(is_v ? hk - kv.n_kv : hk) << kv.page_shift) * hd);
            }
            h0 += kRows * RPW;
            if (h0 >= h_end) break;
            load(h0);
        }
    }
}

template <class T, class TQ, Form FORM>
cudaError_t launch(const PagedAppendArgs &a, const PagedRope &r, void *q_out, int lpr, dim3 grid, int splits, int share,
                   cudaStream_t st) {
    auto go = [&](auto *kern) {
        return launch_pdl(kern, grid, dim3(kThreads), 0, st, a, r, static_cast<TQ *>(q_out), splits, share);
    };
    if (lpr == 8) return go(k_paged_append_rope<T, TQ, 8, FORM>);
    if (lpr == 16) return go(k_paged_append_rope<T, TQ, 16, FORM>);
    return go(k_paged_append_rope<T, TQ, 32, FORM>);
}

}  // namespace

cudaError_t launch_paged_append_rope(const PagedAppendArgs &a, const PagedRope &r, void *q_out, bool q16, int sms, cudaStream_t st) {
    const int rows = a.n_heads + 2 * a.kv.n_kv, hd = a.kv.hd, lpr = hd <= 64 ? 8 : hd <= 128 ? 16 : 32;
    const int batch = kRows * (32 / lpr), batches = (rows + batch - 1) / batch;
    // warps per token: one where that fills the SMs (24 warps each), else as many as there are batches of rows
    const long long want = std::min<long long>(batches, (24ll * sms + a.n_tokens - 1) / a.n_tokens);
    const int share = (batches + static_cast<int>(want) - 1) / static_cast<int>(want) * batch;
    const int splits = (rows + share - 1) / share;
    const long long ctas = (static_cast<long long>(a.n_tokens) * splits + kThreads / 32 - 1) / (kThreads / 32);
    const dim3 grid(static_cast<unsigned>(std::min<long long>(ctas, 32ll * sms)));
    auto al16 = [](const void *p, long long s) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s % 4 == 0; };
    const bool vec = hd % 8 == 0 && (r.interleaved || r.n_dims % 8 == 0) && al16(a.q, a.q_stride) && al16(a.k, a.k_stride) &&
                     al16(a.v, a.v_stride);
    const Form form = !vec ? ODD : r.interleaved ? NEIGHBOURS : r.n_dims == hd ? HALVES : SOME;
    auto of = [&](auto t, auto tq) {
        using T = decltype(t);
        using TQ = decltype(tq);
        switch (form) {
            case HALVES: return launch<T, TQ, HALVES>(a, r, q_out, lpr, grid, splits, share, st);
            case NEIGHBOURS: return launch<T, TQ, NEIGHBOURS>(a, r, q_out, lpr, grid, splits, share, st);
            case SOME: return launch<T, TQ, SOME>(a, r, q_out, lpr, grid, splits, share, st);
            default: return launch<T, TQ, ODD>(a, r, q_out, lpr, grid, splits, share, st);
        }
    };
    if (a.kv.dtype == STYX_F32) return of(float{}, float{});
    if (a.kv.dtype == STYX_F16) return q16 ? of(__half{}, __half{}) : of(__half{}, float{});
    return q16 ? of(__nv_bfloat16{}, __nv_bfloat16{}) : of(__nv_bfloat16{}, float{});
}

}  // namespace styx
