// paged_attn.cu -- attention of one new token per sequence over a paged KV
// cache (styx_paged_attend, include/styx_serve.h).
//
// k_attend_fma.  CTA (an equal share of the tile list, paged_split.cuh): eight
// warps take rows in turn, LPR lanes per row with eight elements each, so that
// q (8 heads x 8 elements) and O stay in registers and K and V are read once
// per eight q heads (with more of them per kv head, once per group of eight).
// A lane copies exactly the bytes that it will use itself (cp.async into a
// ring of its own), so no barrier is needed between copy and use and 128 KB
// or more per SM are in flight.  The 8 heads' dot products are summed over
// the row's lanes by halving exchanges, which leave each lane one head's
// score; maxima move only when a score passes them by 2^8.  A lane has two
// rows at once, whose exchanges overlap.
// Measured (B200): 8 sequences (one empty, two shorter), the last 2048 f32 rows
// of 32 / 4 heads of 128 (52.7 MB) in 22.4 us in a graph over one state, which
// then lies in L2, 25 as called over several.  Of the first, with the finish:
// 2 us until a CTA knows its share, 4 for pages, q and the first copies, 11 of
// rows (issue and exchanges, not memory: 16-bit rows cost as much), 2 for the
// result, 2 for the finish.  One row at a time and tiles of 128 rows: 27 us
// (some CTAs had four times the work of others); pages one by one and q by 4
// bytes: 31 us.
#include <cuda_runtime.h>

#include <cstdint>

#include "paged_split.cuh"

namespace styx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int NH = 8;                 // q heads of a group
constexpr int kPitch = 256;           // floats of a head's O in a portion's result
constexpr int kSets = 2;              // rows of a lane at once: two chains of exchanges in flight
constexpr float kSlack = 8.f;

// LPR lanes per row, 8 elements each: head_dim <= 8 LPR.  f32: two 16-byte
// chunks, at 4 lane and 4 (LPR + lane); 16-bit: one, at 8 lane.
template <class T, int LPR>
struct Lay {
    static constexpr int chunks = sizeof(T) == 4 ? 2 : 1;
    static constexpr int rpw = 32 / LPR;                      // rows of a warp side by side
    static constexpr int set = 2 * chunks * 16 * kThreads;    // bytes of the CTA's rows side by side, K then V
    static constexpr int stage = kSets * set;
    static constexpr int stages = (sizeof(T) == 4 ? 10 : 16) / kSets;   // 160 KB, 128 KB
    __device__ static __forceinline__ int elem(int l, int e) {   // element e of lane l of the row
        return chunks == 2 ? (e < 4 ? 4 * l + e : 4 * (LPR + l) + e - 4) : 8 * l + e;
    }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on) {   // off: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
template <class T>
__device__ __forceinline__ void unpack(const uint8_t *p, float (&v)[8]);
template <>
__device__ __forceinline__ void unpack<float>(const uint8_t *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 16 * kThreads);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint8_t *p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint8_t *p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
// two f32 fused multiply-adds in one instruction
__device__ __forceinline__ void fma2(float2 &d, float2 a, float2 b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;"
        : "+l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)));
}

template <class T, int LPR>
__global__ void __launch_bounds__(kThreads, 1) k_attend_fma(PagedAttendArgs a) {
    using Y = Lay<T, LPR>;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float s_m[kWarps][NH], s_l[kWarps][NH], s_L[NH], s_M[NH];
    const PagedKv &kv = a.kv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = kv.hd;
    const int rl = lane % LPR, rw = lane / LPR;      // lane of the row, row of the warp
    const int groups = (a.gqa + NH - 1) / NH, segs = kv.n_kv * groups;
    pdl_trigger();
    pdl_wait();
    long long T_, G;
    Walk wk;
    share_of(a, segs, blockIdx.x, wk, T_, G);
    // the head whose sum the halving exchanges leave in this lane: from the lane bits LPR/2, LPR/4, LPR/8
    const int myh = ((rl & (LPR / 2)) ? 4 : 0) | ((rl & (LPR / 4)) ? 2 : 0) | ((rl & (LPR / 8)) ? 1 : 0);
    const uint32_t mine = smem_addr(ring) + tid * 16;
    const float l2 = a.scale * 1.4426950408889634f;
    constexpr int SIDE = kWarps * Y::rpw, STEP = kSets * SIDE;   // rows of the CTA side by side; at once

    while (wk.next(a, segs)) {
        const Seq s(a, wk.b, false);
        const int j = wk.seg / groups, g0 = (wk.seg - j * groups) * NH, ng = min(NH, a.gqa - g0);
        const long long h0 = static_cast<long long>(wk.b) * a.n_heads + j * a.gqa + g0;
        const int32_t *table = kv.table + static_cast<long long>(wk.b) * kv.table_stride;
        const int lo = max(s.first, (s.tile0 + wk.t0) << a.tile_shift);
        const int hi = static_cast<int>(min(static_cast<long long>(s.n), static_cast<long long>(s.tile0 + wk.t1) << a.tile_shift));
        const int iters = hi > lo ? (hi - lo + STEP - 1) / STEP : 0;
        const int row0 = lo + warp * Y::rpw + rw;
        float *scores = a.scores + (static_cast<long long>(wk.b) * kv.n_kv + j) *
                                       (static_cast<long long>(kv.max_pages) << kv.page_shift) * a.gqa + g0;
        float2 o[NH][4];
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[h][e] = make_float2(0.f, 0.f);
        float m = kNone, l = 0.f;                    // of head myh, over this lane's rows
        // set n: the lane's row row0 + n SIDE
        auto page_of = [&](int n) {
            const int r = row0 + n * SIDE;
            return r < hi ? ld_now(table + (r >> kv.page_shift)) : -1;
        };
        // copies of set n; returns whether its row is seen
        auto copy = [&](int n, int page) {
            const int r = row0 + n * SIDE;
            const bool in = r < hi, ok = in && static_cast<unsigned>(page) < static_cast<unsigned>(kv.n_pages);
            if (in && !ok && rl == 0) atomicExch(kv.err, kErrBadPos);
            const long long off = ok ? page * kv.page_stride + static_cast<long long>((j << kv.page_shift) +
                                                                                     (r & ((1 << kv.page_shift) - 1))) * hd
                                     : 0;
            const uint32_t dst = mine + (n % (kSets * Y::stages)) * Y::set;
#pragma unroll
            for (int c = 0; c < Y::chunks; c++) {
                const int e = Y::elem(rl, 4 * c);
                const bool on = ok && e < hd;
                copy16(dst + c * 16 * kThreads, static_cast<const T *>(kv.k) + (on ? off + e : 0), on);
                copy16(dst + (Y::chunks + c) * 16 * kThreads, static_cast<const T *>(kv.v) + (on ? off + e : 0), on);
            }
            return ok;
        };
        // the first rows' pages and q, all loads at once, then the first copies
        unsigned seen = 0;                           // bit n % 32: set n's row is seen
        int pages[kSets * Y::stages];
#pragma unroll
        for (int n = 0; n < kSets * Y::stages; n++) pages[n] = page_of(n);
        float2 q[NH][4];
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int c = Y::elem(rl, 4 * i);    // (head_dim is a multiple of 4)
                const float4 v = h < ng && c < hd ? *reinterpret_cast<const float4 *>(a.q + (h0 + h) * hd + c)
                                                  : make_float4(0.f, 0.f, 0.f, 0.f);
                q[h][2 * i] = make_float2(v.x * l2, v.y * l2);
                q[h][2 * i + 1] = make_float2(v.z * l2, v.w * l2);
            }
#pragma unroll
        for (int n = 0; n < kSets * (Y::stages - 1); n++) {
            seen |= static_cast<unsigned>(copy(n, pages[n])) << (n & 31);
            if (n % kSets == kSets - 1) asm volatile("cp.async.commit_group;" ::: "memory");
        }
        int page[kSets];
#pragma unroll
        for (int u = 0; u < kSets; u++) page[u] = pages[kSets * (Y::stages - 1) + u];
        for (int it = 0; it < iters; it++) {
#pragma unroll
            for (int u = 0; u < kSets; u++) {
                const int n = kSets * (it + Y::stages - 1) + u, np = page_of(n + kSets);
                const unsigned bit = 1u << (n & 31);
                seen = copy(n, page[u]) ? seen | bit : seen & ~bit;
                page[u] = np;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(Y::stages - 1) : "memory");
            const uint8_t *st = ring + (it % Y::stages) * Y::stage + tid * 16;
            float x[kSets];
            bool on[kSets], rises = false;
#pragma unroll
            for (int u = 0; u < kSets; u++) {
                float kf[8];
                unpack<T>(st + u * Y::set, kf);
                float d[NH];
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    float2 t = make_float2(0.f, 0.f);
#pragma unroll
                    for (int e = 0; e < 4; e++) fma2(t, q[h][e], make_float2(kf[2 * e], kf[2 * e + 1]));
                    d[h] = t.x + t.y;
                }
                // sums over the row's lanes: eight values halve three times, the rest is one value
                float t4[4], t2[2];
                {
                    const bool up = rl & (LPR / 2);
#pragma unroll
                    for (int i = 0; i < 4; i++) t4[i] = (up ? d[4 + i] : d[i]) + __shfl_xor_sync(0xffffffffu, up ? d[i] : d[4 + i], LPR / 2);
                }
                {
                    const bool up = rl & (LPR / 4);
#pragma unroll
                    for (int i = 0; i < 2; i++) t2[i] = (up ? t4[2 + i] : t4[i]) + __shfl_xor_sync(0xffffffffu, up ? t4[i] : t4[2 + i], LPR / 4);
                }
                {
                    const bool up = rl & (LPR / 8);
                    x[u] = (up ? t2[1] : t2[0]) + __shfl_xor_sync(0xffffffffu, up ? t2[0] : t2[1], LPR / 8);
                }
#pragma unroll
                for (int k = LPR / 16; k; k >>= 1) x[u] += __shfl_xor_sync(0xffffffffu, x[u], k);
                const int n = kSets * it + u, r = row0 + n * SIDE;
                on[u] = (seen >> (n & 31)) & 1;
                if (a.acc_out && r < hi && (rl & (LPR / 8 - 1)) == 0 && myh < ng)
                    scores[static_cast<long long>(r) * a.gqa + myh] = on[u] ? x[u] : -INFINITY;
                rises |= on[u] && x[u] > m + kSlack;
            }
            if (__any_sync(0xffffffffu, rises)) {
                // the warp's maximum of every head; what was summed is rescaled
                float mx = kNone;
#pragma unroll
                for (int u = 0; u < kSets; u++) mx = on[u] ? fmaxf(mx, x[u]) : mx;
#pragma unroll
                for (int k = LPR; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
                mx = fmaxf(m, mx);
                const float f = ex2(m - mx);
                l *= f;
                m = mx;
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    const int src = ((h & 4) ? LPR / 2 : 0) | ((h & 2) ? LPR / 4 : 0) | ((h & 1) ? LPR / 8 : 0);
                    const float fh = __shfl_sync(0xffffffffu, f, src, LPR);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        o[h][e].x *= fh;
                        o[h][e].y *= fh;
                    }
                }
            }
            float p[kSets];
#pragma unroll
            for (int u = 0; u < kSets; u++) {
                p[u] = on[u] ? ex2(x[u] - m) : 0.f;
                l += p[u];
            }
#pragma unroll
            for (int u = 0; u < kSets; u++) {
                float vf[8];
                unpack<T>(st + u * Y::set + Y::chunks * 16 * kThreads, vf);
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    const int src = ((h & 4) ? LPR / 2 : 0) | ((h & 2) ? LPR / 4 : 0) | ((h & 1) ? LPR / 8 : 0);
                    const float ph = __shfl_sync(0xffffffffu, p[u], src, LPR);
#pragma unroll
                    for (int e = 0; e < 4; e++) fma2(o[h][e], make_float2(ph, ph), make_float2(vf[2 * e], vf[2 * e + 1]));
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        // the warp's rows, then the warps, through shared memory
#pragma unroll
        for (int k = LPR; k < 32; k <<= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
        if (rw == 0 && (rl & (LPR / 8 - 1)) == 0) {
            s_m[warp][myh] = m;
            s_l[warp][myh] = l;
        }
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int k = LPR; k < 32; k <<= 1) {
                    o[h][e].x += __shfl_xor_sync(0xffffffffu, o[h][e].x, k);
                    o[h][e].y += __shfl_xor_sync(0xffffffffu, o[h][e].y, k);
                }
        __syncthreads();                             // every warp is done with the ring
        float *so = reinterpret_cast<float *>(ring); // [warps][NH][8 LPR]
        if (rw == 0)
#pragma unroll
            for (int h = 0; h < NH; h++)
#pragma unroll
                for (int e = 0; e < 8; e++) so[(warp * NH + h) * 8 * LPR + Y::elem(rl, e)] = (&o[h][0].x)[e];
        if (tid < NH) {
            float M = kNone, L = 0.f;
            for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_m[w][tid]);
            for (int w = 0; w < kWarps; w++) L += s_l[w][tid] * ex2(s_m[w][tid] - M);
            s_M[tid] = M;
            s_L[tid] = L;
        }
        __syncthreads();
        const bool whole = wk.t0 == 0 && wk.t1 == wk.nt;
        if (wk.t1 == wk.nt && tid == 0) a.cnt[static_cast<long long>(wk.b) * segs + wk.seg] = cut_of(wk, blockIdx.x, T_, G);
        float *part = part_at(a, blockIdx.x, wk.t0 == 0);
        for (int i = tid; i < ng * hd; i += kThreads) {
            const int h = i / hd, c = i - h * hd;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) v += so[(w * NH + h) * 8 * LPR + c] * ex2(s_m[w][h] - s_M[h]);
            if (whole) a.out[(h0 + h) * hd + c] = s_L[h] == 0.f ? 0.f : v / s_L[h];
            else part[h * kPitch + c] = v;
        }
        if (tid < ng) {
            const float M = s_M[tid], L = s_L[tid];
            if (!whole) {
                part[a.part_floats - 32 + tid] = M;
                part[a.part_floats - 16 + tid] = L;
            } else {
                if (a.lse) a.lse[h0 + tid] = lse_of(M, L);
                if (a.acc_out) {
                    a.ml[2 * (h0 + tid)] = M;
                    a.ml[2 * (h0 + tid) + 1] = L;
                }
            }
        }
        __syncthreads();                             // the ring and the sums are free again
    }
}

// ------------------------------------------------------------ finish
// Blocks [0, joins): the O of cut segments.  Head = WPH warps, which share
// its portions; all loads of a warp's up to eight portions are in flight at
// once, so a join costs about two trips to L2 however many portions there
// are.  Blocks from joins on (acc_out): 256 rows of one (sequence, kv head),
//   acc_out[r] = (newest row: 0, else acc[r]) + sum of 2^(score - M) / L,
// with M and L of the group's heads from the portions, as the join has them.
template <int NHG, int NV, int WPH>   // heads of a group; float4s of a head's O per lane; warps per head
__global__ void __launch_bounds__(256) k_attend_finish(PagedAttendArgs a, int joins, int row_blocks) {
    pdl_trigger();
    constexpr int HPC = 8 / WPH;      // heads of a CTA
    __shared__ float4 s_o[8][32 * NV];
    __shared__ float s_M[64], s_L[64];
    const PagedKv &kv = a.kv;
    const int groups = (a.gqa + NHG - 1) / NHG, segs = kv.n_kv * groups;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    if (static_cast<int>(blockIdx.x) < joins) {
        const int at = blockIdx.x / (NHG / HPC), h = (blockIdx.x - at * (NHG / HPC)) * HPC + warp / WPH, w = warp % WPH;
        const unsigned c = ld_cg(a.cnt + at);
        const int np = static_cast<int>(c & 0xFFFFu);
        if (np == 0) return;
        if (static_cast<int>(c >> 16) + np > a.workers) {   // (lengths that changed during the call)
            if (threadIdx.x == 0) atomicExch(kv.err, kErrBadPos);
            return;
        }
        const int b = at / segs, seg = at - b * segs, j = seg / groups, g0 = (seg - j * groups) * NHG;
        const int own0 = static_cast<int>(c >> 16);
        const bool on = h < min(NHG, a.gqa - g0);
        float M = kNone, L = 0.f;
        float4 o[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on)
            for (int i0 = w; i0 < np; i0 += 8 * WPH) {
                float4 x[8][NV];
                float m[8], l[8], top = M;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int k = i0 + i * WPH, p = min(k, np - 1);
                    const float *pp = part_at(a, own0 + p, p == 0);
                    m[i] = ld_cg(pp + a.part_floats - 32 + h);
                    l[i] = ld_cg(pp + a.part_floats - 16 + h);
#pragma unroll
                    for (int v = 0; v < NV; v++) x[i][v] = ld_cg(reinterpret_cast<const float4 *>(pp + h * 128 * NV) + v * 32 + lane);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, m[i]);
                const float f0 = ex2(M - top);
                M = top;
                L *= f0;
#pragma unroll
                for (int v = 0; v < NV; v++) o[v] = make_float4(o[v].x * f0, o[v].y * f0, o[v].z * f0, o[v].w * f0);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (i0 + i * WPH >= np) break;
                    const float f = ex2(m[i] - M);
                    L += f * l[i];
#pragma unroll
                    for (int v = 0; v < NV; v++) {
                        o[v].x += f * x[i][v].x;
                        o[v].y += f * x[i][v].y;
                        o[v].z += f * x[i][v].z;
                        o[v].w += f * x[i][v].w;
                    }
                }
            }
        if constexpr (WPH > 1) {
#pragma unroll
            for (int v = 0; v < NV; v++) s_o[warp][v * 32 + lane] = o[v];
            if (lane == 0) {
                s_M[warp] = M;
                s_L[warp] = L;
            }
            __syncthreads();
            if (w != 0) return;
            const int w0 = warp;
            for (int k = 1; k < WPH; k++) M = fmaxf(M, s_M[w0 + k]);
            L = 0.f;
#pragma unroll
            for (int v = 0; v < NV; v++) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < WPH; k++) {
                const float f = ex2(s_M[w0 + k] - M);
                L += f * s_L[w0 + k];
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    const float4 y = s_o[w0 + k][v * 32 + lane];
                    o[v].x += f * y.x;
                    o[v].y += f * y.y;
                    o[v].z += f * y.z;
                    o[v].w += f * y.w;
                }
            }
        }
        if (!on) return;
        const long long at_h = static_cast<long long>(b) * a.n_heads + j * a.gqa + g0 + h;
        const float r = inverse_sum(L);
#pragma unroll
        for (int v = 0; v < NV; v++)
            if (4 * lane + 128 * v < kv.hd)
                *reinterpret_cast<float4 *>(a.out + at_h * kv.hd + 4 * lane + 128 * v) =
                    make_float4(o[v].x * r, o[v].y * r, o[v].z * r, o[v].w * r);
        if (lane == 0 && a.lse) a.lse[at_h] = lse_of(M, L);
        return;
    }
    // ---------------- accumulated weights
    const int blk = blockIdx.x - joins, bj = blk / row_blocks, b = bj / kv.n_kv, j = bj - b * kv.n_kv;
    const int n = paged_len(kv, b, false), first = a.window > 0 && a.window < n ? n - a.window : 0;
    const long long max_rows = static_cast<long long>(kv.max_pages) << kv.page_shift;
    const float *scores = a.scores + (static_cast<long long>(b) * kv.n_kv + j) * max_rows * a.gqa;
    const long long line = static_cast<long long>(bj) * a.acc_stride;
    for (int r0 = (blk - bj * row_blocks) * 256; r0 < n; r0 += row_blocks * 256) {
        const int r = r0 + threadIdx.x;
        float w = 0.f;
        const float old = r < n - 1 ? a.acc[line + r] : 0.f;
        for (int gc = 0; gc < a.gqa; gc += 64) {     // 64 heads at a time
            const int gn = min(64, a.gqa - gc);
            __syncthreads();
            for (int g = warp; g < gn; g += 8) {
                const int h = gc + g, seg = j * groups + h / NHG, hh = h % NHG;
                const unsigned c = ld_cg(a.cnt + static_cast<long long>(b) * segs + seg);
                const int own0 = static_cast<int>(c >> 16), np = min(static_cast<int>(c & 0xFFFFu), a.workers - own0);
                float M = kNone, L = 0.f;
                if (np == 0) {
                    const float *ml = a.ml + 2 * (static_cast<long long>(b) * a.n_heads + j * a.gqa + h);
                    M = ld_cg(ml);
                    L = ld_cg(ml + 1);
                } else {
                    for (int i = lane; i < np; i += 32) {
                        const float *pp = part_at(a, own0 + i, i == 0);
                        const float m = ld_cg(pp + a.part_floats - 32 + hh), l = ld_cg(pp + a.part_floats - 16 + hh);
                        const float top = fmaxf(M, m);
                        L = L * ex2(M - top) + l * ex2(m - top);
                        M = top;
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) {
                        const float m = __shfl_xor_sync(0xffffffffu, M, o), l = __shfl_xor_sync(0xffffffffu, L, o);
                        const float top = fmaxf(M, m);
                        L = L * ex2(M - top) + l * ex2(m - top);
                        M = top;
                    }
                }
                if (lane == 0) {
                    s_M[g] = M;
                    s_L[g] = inverse_sum(L);
                }
            }
            __syncthreads();
            if (r < n && r >= first) {
                const float *sc = scores + static_cast<long long>(r) * a.gqa + gc;
                int g = 0;
                if ((a.gqa & 3) == 0)
                    for (; g < gn; g += 4) {
                        const float4 x = ld_cg(reinterpret_cast<const float4 *>(sc + g));
                        w += ex2(x.x - s_M[g]) * s_L[g] + ex2(x.y - s_M[g + 1]) * s_L[g + 1] +
                             ex2(x.z - s_M[g + 2]) * s_L[g + 2] + ex2(x.w - s_M[g + 3]) * s_L[g + 3];
                    }
                for (; g < gn; g++) w += ex2(ld_cg(sc + g) - s_M[g]) * s_L[g];
            }
        }
        if (r < n) a.acc_out[line + r] = old + w;
    }
}

template <int NHG, int NV>
cudaError_t finish(const PagedAttendArgs &a, cudaStream_t st) {
    const long long rows = static_cast<long long>(a.kv.max_pages) << a.kv.page_shift;
    const int groups = (a.gqa + NHG - 1) / NHG;
    const long long segs = static_cast<long long>(a.kv.n_seqs) * a.kv.n_kv * groups;
    // nothing is cut where no sequence can have a second tile
    const bool cut = rows > (1ll << a.tile_shift);
    const long long want = (rows + 255) / 256, lines = static_cast<long long>(a.kv.n_seqs) * a.kv.n_kv;
    const int row_blocks = a.acc_out ? static_cast<int>(want < 4096 ? want : 4096) : 0;
    // eight warps per head where that is a wave of CTAs at most (148 SMs x 8), else one
    if (segs * NHG <= 1184) {
        const long long joins = cut ? segs * NHG : 0, grid = joins + row_blocks * lines;
        if (grid == 0) return cudaSuccess;
        return launch_pdl(k_attend_finish<NHG, NV, 8>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, st, a,
                          static_cast<int>(joins), row_blocks);
    }
    const long long joins = cut ? segs * (NHG / 8) : 0, grid = joins + row_blocks * lines;
    if (grid == 0) return cudaSuccess;
    return launch_pdl(k_attend_finish<NHG, NV, 1>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, st, a,
                      static_cast<int>(joins), row_blocks);
}

template <class T, int LPR>
cudaError_t launch(const PagedAttendArgs &a, int grid, cudaStream_t st) {
    constexpr int ring = Lay<T, LPR>::stage * Lay<T, LPR>::stages, join = kWarps * NH * 8 * LPR * 4;
    constexpr int smem = ring > join ? ring : join;
    const cudaError_t e = allow_smem<k_attend_fma<T, LPR>>(smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_attend_fma<T, LPR>, dim3(grid), dim3(kThreads), smem, st, a);
}
template <class T>
cudaError_t launch_t(const PagedAttendArgs &a, int grid, cudaStream_t st) {
    return a.kv.hd <= 64 ? launch<T, 8>(a, grid, st) : a.kv.hd <= 128 ? launch<T, 16>(a, grid, st) : launch<T, 32>(a, grid, st);
}

}  // namespace

int attend_grid(const PagedAttendArgs &a, int nh, int sms) {
    // no more CTAs than tiles there can be
    const long long tiles = static_cast<long long>(a.kv.n_seqs) * a.kv.n_kv * ((a.gqa + nh - 1) / nh) *
                            (((static_cast<long long>(a.kv.max_pages) << a.kv.page_shift) + (1ll << a.tile_shift) - 1) >> a.tile_shift);
    return static_cast<int>(tiles < sms ? tiles : sms);
}

cudaError_t launch_attend_finish(const PagedAttendArgs &a, int nh, int pitch, cudaStream_t st) {
    if (pitch == 256) return finish<8, 2>(a, st);
    return nh == 8 ? finish<8, 1>(a, st) : finish<16, 1>(a, st);
}

uint64_t attend_fma_parts(int sms) { return 2ull * sms * attend_part(NH, kPitch) * 4; }

cudaError_t launch_attend_fma(PagedAttendArgs a, int sms, cudaStream_t st) {
    a.tile_shift = a.kv.hd <= 64 ? 6 : 5;   // the rows that a CTA takes at once (head_dim above 128: twice those)
    a.seg_cost = 3;
    a.part_floats = attend_part(NH, kPitch);
    const int grid = a.workers = attend_grid(a, NH, sms);
    const cudaError_t e = a.kv.dtype == STYX_F16    ? launch_t<__half>(a, grid, st)
                          : a.kv.dtype == STYX_BF16 ? launch_t<__nv_bfloat16>(a, grid, st)
                                                    : launch_t<float>(a, grid, st);
    return e != cudaSuccess ? e : launch_attend_finish(a, NH, kPitch, st);
}

}  // namespace styx
