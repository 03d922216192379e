// paged.cu -- rows into and out of a paged KV cache (include/styx_serve.h):
//
//   k_paged_append   per-head RMSNorm, RoPE and the rounded K / V rows
//   k_paged_evict    the rows that stay, and the moves that close the gaps
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "cluster.cuh"
#include "paged.cuh"

namespace styx {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ------------------------------------------------------------ append
// A CTA takes tokens in turn (blockIdx.y: a share of their rows when tokens
// are few).  The token's cosines and sines are computed once, by the first
// threads, into shared memory: the angle in turns, pos * base^(-2i/d) / 2 pi,
// is held in 64 bits and reduced to a fraction of a turn before it is rounded
// to f32, so its error does not grow with the position.  Then a warp takes
// four of the token's rows (q heads, k heads, v heads) at a time, all loads
// first; lane l holds the pairs (i, i + d/2) of i = 2 l, 2 l + 1 (+ 64).
constexpr int kAppThreads = 256, kAppRows = 4;

template <class T>
__device__ __forceinline__ void store2(T *p, float a, float b) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2 *>(p) = make_float2(a, b);
    } else {
        T v[2] = {from_f<T>(a), from_f<T>(b)};
        *reinterpret_cast<uint32_t *>(p) = *reinterpret_cast<uint32_t *>(v);
    }
}

// K: rounds of 64 pairs, d <= 128 K (d/2 is even: rows are of 16 bytes'
// multiples).  vec: every row of the inputs is 8-byte aligned, else loads are
// by element.
template <class T, int K>
__global__ void __launch_bounds__(kAppThreads) k_paged_append(PagedAppendArgs a, bool vec) {
    pdl_trigger();
    __shared__ float s_cs[2][2][128];
    const PagedKv &kv = a.kv;
    const int hd = kv.hd, half = hd >> 1, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.n_heads + 2 * kv.n_kv;
    const double turn = tid < half ? exp2(a.log2_base * tid) * 0.15915494309189535 : 0.0;   // 1 / 2 pi
    pdl_wait();
    int buf = 0;
    for (int t = blockIdx.x; t < a.n_tokens; t += gridDim.x, buf ^= 1) {
        const int b = a.seq ? __ldg(a.seq + t) : t, pos = __ldg(a.pos + t);
        const bool seq_ok = static_cast<unsigned>(b) < static_cast<unsigned>(kv.n_seqs);
        const int r = !seq_ok ? -1 : a.row ? __ldg(a.row + t) : __ldg(kv.lens + b) - 1;
        bool row_ok = r >= 0 && r < (static_cast<long long>(kv.max_pages) << kv.page_shift);
        const long long off = row_ok ? paged_off(kv, b, 0, r) : -1;   // of kv head 0
        row_ok = off >= 0;
        if (tid == 0 && blockIdx.y == 0 && (!seq_ok || (r >= 0 && !row_ok))) atomicExch(kv.err, kErrBadPos);
        if (tid < half) {
            const double x = pos * turn, f = x - rint(x);
            float s, c;
            sincospif(static_cast<float>(2.0 * f), &s, &c);
            s_cs[buf][0][tid] = c;
            s_cs[buf][1][tid] = s;
        }
        __syncthreads();   // (the other buffer is free again: every warp has passed here once more since it read it)
        for (int h0 = (blockIdx.y * (kAppThreads / 32) + warp) * kAppRows; h0 < rows;
             h0 += gridDim.y * (kAppThreads / 32) * kAppRows) {
            float2 x[kAppRows][K], y[kAppRows][K];
#pragma unroll
            for (int j = 0; j < kAppRows; j++) {
                const int h = h0 + j;
                if (h >= rows) break;
                const float *src = h < a.n_heads             ? a.q + t * a.q_stride + static_cast<long long>(h) * hd
                                   : h < a.n_heads + kv.n_kv ? a.k + t * a.k_stride + static_cast<long long>(h - a.n_heads) * hd
                                                             : a.v + t * a.v_stride + static_cast<long long>(h - a.n_heads - kv.n_kv) * hd;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const int i = 2 * lane + 64 * k;
                    x[j][k] = y[j][k] = make_float2(0.f, 0.f);
                    if (i < half) {
                        if (vec) {
                            x[j][k] = __ldcs(reinterpret_cast<const float2 *>(src + i));
                            y[j][k] = __ldcs(reinterpret_cast<const float2 *>(src + half + i));
                        } else {
                            x[j][k] = make_float2(src[i], src[i + 1]);
                            y[j][k] = make_float2(src[half + i], src[half + i + 1]);
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kAppRows; j++) {
                const int h = h0 + j;
                if (h >= rows) break;
                const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + kv.n_kv;
                const float *w = is_q ? a.q_norm : a.k_norm;
                if (w && !is_v) {
                    float ss = 0.f;
#pragma unroll
                    for (int k = 0; k < K; k++)
                        ss += x[j][k].x * x[j][k].x + x[j][k].y * x[j][k].y + y[j][k].x * y[j][k].x + y[j][k].y * y[j][k].y;
                    const float scale = 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(hd) + a.eps);
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        const int i = 2 * lane + 64 * k;
                        if (i < half) {
                            x[j][k].x *= scale * __ldg(w + i);
                            x[j][k].y *= scale * __ldg(w + i + 1);
                            y[j][k].x *= scale * __ldg(w + half + i);
                            y[j][k].y *= scale * __ldg(w + half + i + 1);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const int i = 2 * lane + 64 * k;
                    if (i >= half) continue;
                    float2 u = x[j][k], v = y[j][k];
                    if (!is_v) {
                        const float2 c = *reinterpret_cast<const float2 *>(&s_cs[buf][0][i]);
                        const float2 s = *reinterpret_cast<const float2 *>(&s_cs[buf][1][i]);
                        u = make_float2(x[j][k].x * c.x - y[j][k].x * s.x, x[j][k].y * c.y - y[j][k].y * s.y);
                        v = make_float2(x[j][k].x * s.x + y[j][k].x * c.x, x[j][k].y * s.y + y[j][k].y * c.y);
                    }
                    if (is_q) {
                        if (r < 0) u = v = make_float2(0.f, 0.f);   // padding, or an empty slot
                        float *o = a.q_out + (static_cast<long long>(t) * a.n_heads + h) * hd;
                        store2(o + i, u.x, u.y);
                        store2(o + half + i, v.x, v.y);
                    } else if (row_ok) {
                        const int head = h - a.n_heads - (is_v ? kv.n_kv : 0);
                        T *o = static_cast<T *>(is_v ? kv.v : kv.k) + off + (static_cast<long long>(head) << kv.page_shift) * hd;
                        store2(o + i, u.x, u.y);
                        store2(o + half + i, v.x, v.y);
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------ eviction
constexpr int kEvThreads = 512, kEvWarps = kEvThreads / 32;
constexpr int kEvSlice = 40960;   // keys that a CTA holds in shared memory

// order of the weights as unsigned integers, larger first: protected rows
// above all, NaN as -inf, -0 as +0
__device__ __forceinline__ uint32_t evict_key(float acc, int pos, int next_pos, int n_recent, int n_sink) {
    if (static_cast<long long>(pos) >= static_cast<long long>(next_pos) - n_recent || pos < n_sink) return 0xFFFFFFFFu;
    if (acc != acc) acc = -INFINITY;
    const uint32_t b = __float_as_uint(acc + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);   // +inf: 0xFF800000, below the protected rows' key
}

// what a cluster's CTAs write into each other
struct EvictShared {
    unsigned cnt[2][16][8];                      // [buffer][CTA][threshold]
    unsigned ties[16], holes[16], movers[16];
    unsigned w[2][kEvWarps][8], scan[kEvWarps];
};

// exclusive prefix over the CTA, and the total
__device__ __forceinline__ unsigned cta_scan(unsigned v, unsigned *sh, unsigned &tot) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    unsigned s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 31) sh[w] = s;
    __syncthreads();
    unsigned x = lane < kEvWarps ? sh[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
    }
    tot = __shfl_sync(0xffffffffu, x, 31);
    const unsigned before = __shfl_sync(0xffffffffu, x, w ? w - 1 : 0);
    return (w ? before : 0) + s - v;
}

// A cluster of C CTAs per line (sequence, kv head), each with a slice of its
// rows, whose keys stay in shared memory (STAGED; else they are made again
// from L2 each time).  The key of the budget-th row is found eightfold: seven
// thresholds are counted at once, 11 rounds for 32 bits, one barrier each; no
// atomics, so equal weights cost nothing extra.  Then rows are numbered in
// order: who stays (keys above the threshold, the first rows at it), the
// places below the budget that become free, the rows beyond it that stay;
// the i-th of these moves into the i-th place.  Sources lie at or beyond the
// budget, places below it, so no row is both.
template <bool STAGED>
__global__ void __launch_bounds__(kEvThreads) k_paged_evict(PagedEvictArgs a, int C, int row_bytes) {
    extern __shared__ uint32_t keys[];
    __shared__ EvictShared sh;
    pdl_trigger();
    const PagedKv &kv = a.kv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0, line_no = blockIdx.x / C;
    const int b = line_no / kv.n_kv, j = line_no - b * kv.n_kv;
    auto all_sync = [&] {
        if (C > 1) {
            cl_arrive();
            cl_wait();
        } else {
            __syncthreads();
        }
    };
    auto tell = [&](unsigned *slot, unsigned v, int to) {   // into CTA `to`'s copy of slot
        if (C > 1) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cl_map(smem_addr(slot), to)), "r"(v) : "memory");
        else *slot = v;
    };
    if (C > 1) cl_arrive_relaxed();   // the others have started: waited for before the first store to them
    pdl_wait();
    const int n = paged_len(kv, b, tid == 0 && j == 0 && rank == 0);
    const int left = min(n, a.budget);
    const long long line = static_cast<long long>(line_no) * a.stride;
    const float *acc = a.acc + line;
    const int32_t *pos = a.pos + line;
    if (j == 0 && tid == 0 && rank == 0) a.lens_out[b] = left;
    const int slice = (((n + C - 1) / C) + 3) & ~3, lo = min(n, rank * slice), hi = min(n, lo + slice), len = hi - lo;
    if (C > 1) cl_wait();
    if (n <= a.budget) {   // all stay (every CTA of the cluster comes here)
        for (int r = lo + tid; r < hi; r += kEvThreads) {
            a.acc_out[line + r] = acc[r];
            a.pos_out[line + r] = pos[r];
        }
        return;
    }
    const int np = __ldg(a.next_pos + b);
    if (STAGED) {
#pragma unroll 4
        for (int i = tid; i < len; i += kEvThreads) keys[i] = evict_key(acc[lo + i], pos[lo + i], np, a.n_recent, a.n_sink);
        __syncthreads();
    }
    auto key_at = [&](int i) { return STAGED ? keys[i] : evict_key(acc[lo + i], pos[lo + i], np, a.n_recent, a.n_sink); };
    // ---------------- threshold: at least `left` keys are >= t0, fewer are >= t1
    unsigned long long t0 = 0, t1 = 1ull << 32;
    unsigned above = 0;                                    // keys >= t1
    for (int buf = 0; t1 - t0 > 1; buf ^= 1) {
        const unsigned long long w = t1 - t0;
        unsigned th[7], c[7];
#pragma unroll
        for (int i = 0; i < 7; i++) {
            th[i] = static_cast<unsigned>(t0 + (w * (i + 1)) / 8);
            c[i] = 0;
        }
        for (int i = tid; i < len; i += kEvThreads) {
            const uint32_t k = key_at(i);
#pragma unroll
            for (int z = 0; z < 7; z++) c[z] += k >= th[z];
        }
        unsigned mine = 0;
#pragma unroll
        for (int z = 0; z < 7; z++) {
            const unsigned s = __reduce_add_sync(0xffffffffu, c[z]);
            if (lane == z) mine = s;
        }
        if (lane < 7) sh.w[buf][warp][lane] = mine;
        __syncthreads();
        // lane z of every warp: the CTA's count of threshold z
        unsigned tot = 0;
        if (lane < 7)
#pragma unroll
            for (int q = 0; q < kEvWarps; q++) tot += sh.w[buf][q][lane];
        if (C > 1) {
            if (warp < C && lane < 7) tell(&sh.cnt[buf][rank][lane], tot, warp);
            all_sync();
            tot = 0;
            if (lane < 7)
                for (int q = 0; q < C; q++) tot += sh.cnt[buf][q][lane];
        }
        // thresholds rise, counts fall: the last that still reaches `left`
        const unsigned reach = __ballot_sync(0xffffffffu, lane < 7 && tot >= static_cast<unsigned>(left));
        const int z = __popc(reach) - 1;
        const unsigned long long n0 = t0 + (w * (z + 1)) / 8, n1 = t0 + (w * (z + 2)) / 8;
        if (z < 6) above = __shfl_sync(0xffffffffu, tot, z + 1);
        t1 = z < 6 ? n1 : t1;
        t0 = z < 0 ? t0 : n0;
    }
    const uint32_t thr = static_cast<uint32_t>(t0);
    const unsigned ties = static_cast<unsigned>(left) - above;   // of the rows at thr, the first `ties` stay
    // ---------------- numbering, in row order: ties, then places and movers
    unsigned n_ties = 0;
    for (int i = tid; i < len; i += kEvThreads) n_ties += key_at(i) == thr;
    unsigned tot;
    cta_scan(n_ties, sh.scan, tot);
    if (tid < C) tell(&sh.ties[rank], tot, tid);
    all_sync();
    unsigned tie0 = 0;
    for (int q = 0; q < rank; q++) tie0 += sh.ties[q];
    // pass 0 counts this slice's places and movers, pass 1 lists them
    unsigned hole0 = 0, mover0 = 0;
    for (int pass = 0; pass < 2; pass++) {
        unsigned t_run = tie0, h_run = hole0, m_run = mover0;
        for (int base = 0; base < len; base += kEvThreads) {
            const int i = base + tid, r = lo + i;
            const bool in = i < len;
            const uint32_t k = in ? key_at(i) : 0u;
            const unsigned tr = cta_scan(in && k == thr, sh.scan, tot);
            const bool stay = in && (k > thr || (k == thr && t_run + tr < ties));
            t_run += tot;
            const bool hole = in && r < left && !stay, mover = in && r >= left && stay;
            // (a tile's places and movers in one scan: counts below 2^16)
            const unsigned hm = cta_scan((hole ? 1u : 0u) | (mover ? 1u << 16 : 0u), sh.scan, tot);
            if (pass == 1) {
                int32_t *lists = a.places + static_cast<long long>(line_no) * a.budget;
                if (hole) lists[h_run + (hm & 0xFFFFu)] = r;
                if (mover) (a.src + static_cast<long long>(line_no) * a.budget)[m_run + (hm >> 16)] = r;
                if (in && r < left && stay) {
                    a.acc_out[line + r] = acc[r];
                    a.pos_out[line + r] = pos[r];
                }
            }
            h_run += tot & 0xFFFFu;
            m_run += tot >> 16;
        }
        if (pass == 0) {
            if (tid < C) {
                tell(&sh.holes[rank], h_run, tid);
                tell(&sh.movers[rank], m_run, tid);
            }
            all_sync();
            for (int q = 0; q < rank; q++) {
                hole0 += sh.holes[q];
                mover0 += sh.movers[q];
            }
        }
    }
    all_sync();   // the lists are complete (and visible: release and acquire at cluster scope)
    unsigned moves = 0;
    for (int q = 0; q < C; q++) moves += sh.movers[q];
    // ---------------- moves: a row's K and V by 16-byte pieces, half a warp each where they are 256 bytes
    const int32_t *from_l = a.src + static_cast<long long>(line_no) * a.budget;
    const int32_t *to_l = a.places + static_cast<long long>(line_no) * a.budget;
    const int pieces = row_bytes / 16, size = row_bytes / kv.hd;
    for (unsigned i0 = (rank * kEvWarps + warp) * 4; i0 < moves; i0 += C * kEvWarps * 4) {
        long long from[4], to[4];
#pragma unroll
        for (int z = 0; z < 4; z++) {
            from[z] = to[z] = -1;
            if (i0 + z < moves) {
                const int s = __ldcg(from_l + i0 + z), d = __ldcg(to_l + i0 + z);
                if (lane == 0) {
                    a.acc_out[line + d] = acc[s];
                    a.pos_out[line + d] = pos[s];
                }
                from[z] = paged_off(kv, b, j, s);
                to[z] = paged_off(kv, b, j, d);
                if ((from[z] < 0 || to[z] < 0) && lane == 0) atomicExch(kv.err, kErrBadPos);
            }
        }
        for (int p = lane; p < 2 * pieces; p += 32) {
            char *pool = static_cast<char *>(p < pieces ? kv.k : kv.v);
            const int at = (p < pieces ? p : p - pieces) * 16;
            uint4 v[4];
#pragma unroll
            for (int z = 0; z < 4; z++)
                if (from[z] >= 0 && to[z] >= 0) v[z] = *reinterpret_cast<const uint4 *>(pool + from[z] * size + at);
#pragma unroll
            for (int z = 0; z < 4; z++)
                if (from[z] >= 0 && to[z] >= 0) *reinterpret_cast<uint4 *>(pool + to[z] * size + at) = v[z];
        }
    }
    if (C > 1) all_sync();   // no CTA leaves while another reads its counts
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs &a, int sms, cudaStream_t st) {
    const int rows = a.n_heads + 2 * a.kv.n_kv, per = kAppThreads / 32 * kAppRows;
    // few tokens: their rows over several CTAs; many: eight CTAs per SM take them in turn
    const int parts = std::max(1, std::min((rows + per - 1) / per, 2 * sms / a.n_tokens));
    const dim3 grid(static_cast<unsigned>(std::min(a.n_tokens, 8 * sms)), static_cast<unsigned>(parts));
    auto al8 = [](const void *p, long long s) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0 && s % 2 == 0; };
    const bool vec = al8(a.q, a.q_stride) && al8(a.k, a.k_stride) && al8(a.v, a.v_stride);
    const bool two = a.kv.hd > 128;
    const dim3 block(kAppThreads);
    if (a.kv.dtype == STYX_F16)
        return two ? launch_pdl(k_paged_append<__half, 2>, grid, block, 0, st, a, vec) : launch_pdl(k_paged_append<__half, 1>, grid, block, 0, st, a, vec);
    if (a.kv.dtype == STYX_BF16)
        return two ? launch_pdl(k_paged_append<__nv_bfloat16, 2>, grid, block, 0, st, a, vec)
                   : launch_pdl(k_paged_append<__nv_bfloat16, 1>, grid, block, 0, st, a, vec);
    return two ? launch_pdl(k_paged_append<float, 2>, grid, block, 0, st, a, vec) : launch_pdl(k_paged_append<float, 1>, grid, block, 0, st, a, vec);
}

cudaError_t launch_paged_evict(const PagedEvictArgs &a, cudaStream_t st) {
    const long long rows = static_cast<long long>(a.kv.max_pages) << a.kv.page_shift;
    int C = 1;
    while (C < 8 && rows > 4096ll * C) C <<= 1;
    const long long slice = ((rows + C - 1) / C + 3) & ~3ll;
    const bool staged = slice <= kEvSlice;
    const int row_bytes = a.kv.hd * (a.kv.dtype == STYX_F32 ? 4 : 2);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.kv.n_seqs) * a.kv.n_kv * C);
    cfg.blockDim = dim3(kEvThreads);
    cfg.dynamicSmemBytes = staged ? static_cast<size_t>(slice) * 4 : 0;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = C > 1 ? 2 : 1;
    if (!staged) return cudaLaunchKernelEx(&cfg, k_paged_evict<false>, a, C, row_bytes);
    const cudaError_t e = cudaFuncSetAttribute(k_paged_evict<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvSlice * 4);
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, k_paged_evict<true>, a, C, row_bytes);
}

}  // namespace styx
