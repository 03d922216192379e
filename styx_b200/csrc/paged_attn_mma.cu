// paged_attn_mma.cu -- attention of one new token per sequence over a paged
// f16 / bf16 KV cache on the tensor cores (styx_paged_attend, head_dim up to
// 128, pages of 16 rows or more).
//
// Per kv head the step is two products whose long side is the rows:
//   S^T = K Q^T     [rows x heads],     O^T = V^T P^T     [head_dim x heads]
// with 16 rows (16 elements of head_dim) as M of mma.m16n8k16 and eight q
// heads as N: K and V are the A operands as they lie in memory, nothing is
// padded to a query tile, and eight heads of a kv head cost half of what
// they would as rows.  The kernel's time is HBM's: 512 bytes a row (16 bits,
// head_dim 128) against 6 N-tiles of 8 MMAs.
//
// Precision.  q and p are f32 while K and V have 8 (bf16) or 11 (f16)
// significant bits, so q and p are split into 3 or 2 terms of the cache's
// type that add up to 24 / 22 bits; products are exact, sums f32.
//
// A warp takes 16 rows at a time for itself: its copies (cp.async, 4 KB of K
// and 4 KB of V, contiguous in the page) go round a ring of its own, three
// deep, so that no warp waits for another between a portion's ends and 128 KB
// or more per SM are in flight.  The maximum a row is measured against moves
// only when a score passes it by 2^8.  The next portion's first copies are
// issued before the last one's result is joined from the eight warps.
#include <cuda_runtime.h>

#include <cstdint>

#include "paged_split.cuh"

namespace styx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 16;                      // rows of a warp at once
constexpr int kBuf = kRows * 256;              // K or V of them, 256-byte rows (head_dim 128)
constexpr int kStage = 2 * kBuf, kStages = 3;
constexpr int kRing = kWarps * kStages * kStage;
constexpr int kPad = 132;                      // floats of a head's O in the join: no two heads on one bank
constexpr int kJoin = kWarps * 8 * kPad * 4;   // eight heads of every warp
constexpr float kSlack = 8.f;                  // log2 units a score may pass the maximum by

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on) {   // off: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // of the 8 x 8 matrix that the warp holds
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// a pair of values (low half: x) as sums of terms of the cache's type, largest
// first.  bf16: the f32's 24 significant bits cut into 8 + 8 + 8, exactly;
// f16: rounded to 11, the rest rounded to 11.
template <bool BF>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&t)[BF ? 3 : 2]) {
    if constexpr (BF) {
        uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
#pragma unroll
        for (int i = 0; i < 3; i++) {
            t[i] = __byte_perm(a, b, 0x7632);
            const uint32_t c = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xFFFF0000u));
            const uint32_t d = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xFFFF0000u));
            a = c;
            b = d;
        }
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
        t[0] = *reinterpret_cast<const uint32_t *>(&h);
        t[1] = *reinterpret_cast<const uint32_t *>(&l);
    }
}

// a portion of the CTA's share: its rows [lo, hi) of one segment
struct Part {
    int b, j, g0, ng, lo, hi, base, iters;   // base: lo rounded down to 16
    long long h0;
    const int32_t *table;
    __device__ __forceinline__ void set(const PagedAttendArgs &a, const Walk &wk, int groups, int nh) {
        const Seq s(a, wk.b, false);
        b = wk.b;
        j = wk.seg / groups;
        g0 = (wk.seg - j * groups) * nh;
        ng = min(nh, a.gqa - g0);
        h0 = static_cast<long long>(b) * a.n_heads + j * a.gqa + g0;
        table = a.kv.table + static_cast<long long>(b) * a.kv.table_stride;
        lo = max(s.first, (s.tile0 + wk.t0) * kTile);
        hi = min(s.n, (s.tile0 + wk.t1) * kTile);
        base = lo & ~(kRows - 1);
        iters = hi > lo ? (hi - base + kRows * kWarps - 1) / (kRows * kWarps) : 0;
    }
};

// NT: eights of q heads of a group
template <bool BF, int NT>
__global__ void __launch_bounds__(kThreads, 1) k_attend_mma(PagedAttendArgs a) {
    constexpr int TERMS = BF ? 3 : 2, NH = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_m[kWarps][NH], s_l[kWarps][NH], s_M[NH], s_L[NH];
    const PagedKv &kv = a.kv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = kv.hd;
    const int lr = lane >> 2, lc = lane & 3;   // of the fragments: row (B: column), pair of columns
    const int groups = (a.gqa + NH - 1) / NH, segs = kv.n_kv * groups, ksteps = (hd + 15) / 16, chunks = hd / 8;
    long long T, G;
    Walk wk;
    pdl_trigger();
    pdl_wait();
    share_of<kThreads>(a, segs, *reinterpret_cast<Share<kThreads> *>(smem), wk, T, G);
    __syncthreads();                  // what it left in the ring is read
    const uint32_t ring = smem_addr(smem) + warp * kStages * kStage;
    float *so = reinterpret_cast<float *>(smem + kRing);
    const float l2 = a.scale * 1.4426950408889634f;   // scores in units of log2

    // a tile's page: of its sixteen rows; -1: none
    auto page_of = [&](const Part &p, int it) {
        const int r = p.base + (it * kWarps + warp) * kRows;
        return it < p.iters && r < p.hi ? ld_now(p.table + (r >> kv.page_shift)) : -1;
    };
    // copies of tile `it` of p into slot; what lies outside [lo, hi) or in a page outside the pool is zeros
    auto issue = [&](const Part &p, int it, int page, int slot) {
        const int r0 = p.base + (it * kWarps + warp) * kRows;
        const bool some = it < p.iters && r0 < p.hi, ok = static_cast<unsigned>(page) < static_cast<unsigned>(kv.n_pages);
        if (some) {
            if (!ok && lane == 0) atomicExch(kv.err, kErrBadPos);
            const long long at = ok ? page * kv.page_stride + static_cast<long long>((p.j << kv.page_shift) +
                                                                                     (r0 & ((1 << kv.page_shift) - 1))) * hd
                                    : 0;
            const uint8_t *k = static_cast<const uint8_t *>(kv.k) + at * 2, *v = static_cast<const uint8_t *>(kv.v) + at * 2;
            const int c = lane & 15;
#pragma unroll
            for (int i = 0; i < kRows / 2; i++) {
                const int r = 2 * i + (lane >> 4);
                const bool on = ok && c < chunks && r0 + r >= p.lo && r0 + r < p.hi;
                const uint32_t dst = ring + slot * kStage + r * 256 + ((c ^ (r & 7)) << 4);
                const int src = on ? r * hd * 2 + c * 16 : 0;
                copy16(dst, k + src, on);
                copy16(dst + kBuf, v + src, on);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return some && ok;
    };

    Part P;
    bool have = wk.next(a, segs);
    int slot = 0;                     // of the portion's next tile
    unsigned seen = 0;                // bit s: slot s holds rows that are seen
    int page = -1;
    auto start = [&] {                // a portion's first copies
        P.set(a, wk, groups, NH);
        page = page_of(P, 0);
        int s = slot;
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) {
            const int nx = page_of(P, i + 1);
            const bool on = issue(P, i, page, s);
            seen = on ? seen | (1u << s) : seen & ~(1u << s);
            page = nx;
            s = s + 1 == kStages ? 0 : s + 1;
        }
    };
    if (have) start();
    while (have) {
        // ---------------- q as B fragments, in terms.  f16 has few exponents: a head's largest |q| is brought to
        // [2^9, 2^10), and fh says what its column of S is in units of its terms
        uint32_t qf[NT][8][TERMS][2];
        float fh[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int h = 8 * nt + lr;
            const float *q = a.q + (P.h0 + h) * hd + 2 * lc;
            float2 v[8][2];
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d = 16 * k + 8 * i;
                    v[k][i] = make_float2(0.f, 0.f);
                    if (h < P.ng && d < hd) {
                        const float2 x = *reinterpret_cast<const float2 *>(q + d);
                        v[k][i] = make_float2(x.x * l2, x.y * l2);
                    }
                    mx = fmaxf(mx, fmaxf(fabsf(v[k][i].x), fabsf(v[k][i].y)));
                }
            float up = 1.f, down = 1.f;
            if constexpr (!BF) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int e = max(-110, min(110, static_cast<int>(__float_as_uint(mx) >> 23) - 127 - 9));
                up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                down = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            }
            fh[nt][0] = __shfl_sync(0xffffffffu, down, 8 * lc);        // heads 2 lc, 2 lc + 1 of the eight
            fh[nt][1] = __shfl_sync(0xffffffffu, down, 8 * lc + 4);
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t t[TERMS];
                    split2<BF>(v[k][i].x * up, v[k][i].y * up, t);
#pragma unroll
                    for (int z = 0; z < TERMS; z++) qf[nt][k][z][i] = t[z];
                }
        }
        float m[NT][2], l[NT][2], o[8][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = kNone;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int t = 0; t < 8; t++) o[t][nt][0] = o[t][nt][1] = o[t][nt][2] = o[t][nt][3] = 0.f;
        }
        float *scores = a.scores + (static_cast<long long>(P.b) * kv.n_kv + P.j) *
                                       (static_cast<long long>(kv.max_pages) << kv.page_shift) * a.gqa + P.g0 + 2 * lc;
        for (int it = 0; it < P.iters; it++) {
            {   // the tile kStages - 1 ahead, into the slot of the last one (which every lane has read)
                __syncwarp();
                const int nx = page_of(P, it + kStages), s = slot == 0 ? kStages - 1 : slot - 1;
                const bool on = issue(P, it + kStages - 1, page, s);
                seen = on ? seen | (1u << s) : seen & ~(1u << s);
                page = nx;
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
            __syncwarp();
            const uint32_t kt = ring + slot * kStage, vt = kt + kBuf;
            const bool live = (seen >> slot) & 1;
            slot = slot + 1 == kStages ? 0 : slot + 1;
            const int r0 = P.base + (it * kWarps + warp) * kRows;
            if (!live) {
                // no row of it is seen: past the end, or in a page outside the pool
                if (a.acc_out && r0 < P.hi)
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        for (int h = 0; h < NH; h++)
                            if ((h & 7) >> 1 == lc && h < P.ng && r0 + lr + 8 * i >= P.lo && r0 + lr + 8 * i < P.hi)
                                scores[static_cast<long long>(r0 + lr + 8 * i) * a.gqa + h - 2 * lc] = -INFINITY;
                continue;
            }
            // ---------------- S^T: row lr (+ 8), heads 2 lc, + 1
            float s[NT][TERMS][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int z = 0; z < TERMS; z++) s[nt][z][0] = s[nt][z][1] = s[nt][z][2] = s[nt][z][3] = 0.f;
            {
                const int row = lane & 15;
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (k < ksteps) {
                        uint32_t A[4];
                        ldm4(kt + row * 256 + (((2 * k + (lane >> 4)) ^ (row & 7)) << 4), A);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int z = 0; z < TERMS; z++) mma<BF>(s[nt][z], A, qf[nt][k][z][0], qf[nt][k][z][1]);
                    }
            }
            const bool on[2] = {r0 + lr >= P.lo && r0 + lr < P.hi, r0 + lr + 8 >= P.lo && r0 + lr + 8 < P.hi};
            float x[NT][4];                    // (row lr: heads 0, 1; row lr + 8: heads 0, 1)
            bool up = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float y = s[nt][0][i] + s[nt][1][i];
                    if constexpr (TERMS == 3) y = s[nt][0][i] + (s[nt][1][i] + s[nt][TERMS - 1][i]);
                    x[nt][i] = on[i >> 1] ? (BF ? y : y * fh[nt][i & 1]) : -INFINITY;
                    up |= x[nt][i] > m[nt][i & 1] + kSlack;
                }
            if (a.acc_out)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (on[i]) {
                        float *sc = scores + static_cast<long long>(r0 + lr + 8 * i) * a.gqa;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            if (8 * nt + 2 * lc < P.ng) sc[8 * nt] = x[nt][2 * i];
                            if (8 * nt + 2 * lc + 1 < P.ng) sc[8 * nt + 1] = x[nt][2 * i + 1];
                        }
                    }
            if (__any_sync(0xffffffffu, up)) {
                // new maxima over the sixteen rows; what was summed against the old ones is rescaled
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float v = fmaxf(x[nt][e], x[nt][2 + e]);
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                        v = fmaxf(v, m[nt][e]);
                        const float f = ex2(m[nt][e] - v);
                        m[nt][e] = v;
                        l[nt][e] *= f;
#pragma unroll
                        for (int t = 0; t < 8; t++) {
                            o[t][nt][e] *= f;
                            o[t][nt][2 + e] *= f;
                        }
                    }
            }
            // ---------------- P^T as B fragments: eight rows by eight heads, transposed across the warp
            uint32_t pf[NT][TERMS][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float p0 = on[i] ? ex2(x[nt][2 * i] - m[nt][0]) : 0.f, p1 = on[i] ? ex2(x[nt][2 * i + 1] - m[nt][1]) : 0.f;
                    l[nt][0] += p0;
                    l[nt][1] += p1;
                    uint32_t t[TERMS];
                    // f16: p up to 2^8 is carried as p * 2^7, so that the second term of a small p keeps its bits
                    split2<BF>(BF ? p0 : p0 * 128.f, BF ? p1 : p1 * 128.f, t);
#pragma unroll
                    for (int z = 0; z < TERMS; z++) pf[nt][z][i] = transposed(t[z]);
                }
            // ---------------- O^T += V^T P^T
            {
                const int row = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
                for (int t = 0; t < 8; t++)
                    if (t < ksteps) {
                        uint32_t A[4];
                        ldm4t(vt + row * 256 + (((2 * t + half) ^ (row & 7)) << 4), A);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int z = 0; z < TERMS; z++) mma<BF>(o[t][nt], A, pf[nt][z][0], pf[nt][z][1]);
                    }
            }
        }
        // ---------------- the portion's end: the next one's first copies, then the warps' results joined
        const Part D = P;
        const bool first = wk.t0 == 0, whole = first && wk.t1 == wk.nt;
        if (wk.t1 == wk.nt && tid == 0) a.cnt[static_cast<long long>(wk.b) * segs + wk.seg] = cut_of(wk, T, G);
        have = wk.next(a, segs);
        __syncwarp();
        if (have) start();
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float v = l[nt][e];
                v += __shfl_xor_sync(0xffffffffu, v, 4);
                v += __shfl_xor_sync(0xffffffffu, v, 8);
                v += __shfl_xor_sync(0xffffffffu, v, 16);
                if (lr == 0) {
                    s_m[warp][8 * nt + 2 * lc + e] = m[nt][e];
                    s_l[warp][8 * nt + 2 * lc + e] = v;
                }
            }
        float *part = part_at(a, blockIdx.x, first);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {   // eight heads at a time
#pragma unroll
            for (int t = 0; t < 8; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    so[(warp * 8 + 2 * lc + (i & 1)) * kPad + 16 * t + lr + 8 * (i >> 1)] = BF ? o[t][nt][i] : o[t][nt][i] * 0x1p-7f;
            __syncthreads();
            if (nt == 0) {
                if (tid < NH) {
                    float M = kNone, L = 0.f;
                    for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_m[w][tid]);
                    for (int w = 0; w < kWarps; w++) {
                        const float f = ex2(s_m[w][tid] - M);
                        L += s_l[w][tid] * f;
                        s_m[w][tid] = f;
                    }
                    s_M[tid] = M;
                    s_L[tid] = L;
                }
                __syncthreads();
            }
            for (int i = tid; i < 8 * hd; i += kThreads) {
                const int g = i / hd, c = i - g * hd, h = 8 * nt + g;
                if (h >= D.ng) break;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) v += so[(w * 8 + g) * kPad + c] * s_m[w][h];
                if (whole) a.out[(D.h0 + h) * hd + c] = s_L[h] > 0.f ? v / s_L[h] : 0.f;
                else part[h * 128 + c] = v;
            }
            if (nt + 1 < NT) __syncthreads();
        }
        if (tid < D.ng) {
            const float M = s_M[tid], L = s_L[tid];
            if (!whole) {
                part[kAttendPart - 32 + tid] = M;
                part[kAttendPart - 16 + tid] = L;
            } else {
                if (a.lse) a.lse[D.h0 + tid] = L > 0.f ? M * 0.6931471805599453f + logf(L) : -INFINITY;
                if (a.acc_out) {
                    a.ml[2 * (D.h0 + tid)] = M;
                    a.ml[2 * (D.h0 + tid) + 1] = L;
                }
            }
        }
        __syncthreads();                        // the join's buffers are free again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <bool BF, int NT>
cudaError_t launch(const PagedAttendArgs &a, cudaStream_t st) {
    constexpr int smem = kRing + kJoin;
    const cudaError_t e = allow_smem<k_attend_mma<BF, NT>>(smem);
    if (e != cudaSuccess) return e;
    const cudaError_t e2 = launch_pdl(k_attend_mma<BF, NT>, dim3(a.ctas), dim3(kThreads), smem, st, a);
    return e2 != cudaSuccess ? e2 : launch_attend_finish(a, 8 * NT, 128, st);
}

}  // namespace

cudaError_t launch_attend_mma(PagedAttendArgs a, int sms, cudaStream_t st) {
    const int nt = a.gqa <= 8 ? 1 : 2;
    a.ctas = attend_grid(a, 8 * nt, sms);
    if (a.kv.dtype == STYX_BF16) return nt == 1 ? launch<true, 1>(a, st) : launch<true, 2>(a, st);
    return nt == 1 ? launch<false, 1>(a, st) : launch<false, 2>(a, st);
}

}  // namespace styx
