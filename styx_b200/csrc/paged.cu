// paged.cu -- rows into and out of a paged KV cache (include/styx_serve.h):
//
//   k_paged_append   per-head RMSNorm, RoPE and the rounded K / V rows
//   k_evict_select   the rows that stay, and the moves that close the gaps
//   k_evict_move     K, V, weight and position of the rows that move
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
        const int b = a.seq ? ld_now(a.seq + t) : t, pos = ld_now(a.pos + t);
        const bool seq_ok = static_cast<unsigned>(b) < static_cast<unsigned>(kv.n_seqs);
        const int r = !seq_ok ? -1 : a.row ? ld_now(a.row + t) : ld_now(kv.lens + b) - 1;
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
                            x[j][k] = *reinterpret_cast<const float2 *>(src + i);
                            y[j][k] = *reinterpret_cast<const float2 *>(src + half + i);
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
                            x[j][k].x *= scale * ld_now(w + i);
                            x[j][k].y *= scale * ld_now(w + i + 1);
                            y[j][k].x *= scale * ld_now(w + half + i);
                            y[j][k].y *= scale * ld_now(w + half + i + 1);
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
constexpr int kEvSlice = 40960;               // keys that a CTA holds in shared memory
constexpr int kEvBins = 2048, kEvShare = 4;   // steps of a round; of a thread

// order of the weights as unsigned integers, larger first: protected rows
// above all, NaN as -inf, -0 as +0
constexpr uint32_t kProtected = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t evict_key(float acc, int pos, int next_pos, int n_recent, int n_sink) {
    if (static_cast<long long>(pos) >= static_cast<long long>(next_pos) - n_recent || pos < n_sink) return kProtected;
    if (acc != acc) acc = -INFINITY;
    const uint32_t b = __float_as_uint(acc + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);   // +inf: 0xFF800000, below the protected rows' key
}

struct EvictShared {
    __align__(16) unsigned hist[kEvBins];
    unsigned scan[kEvWarps], red[3][kEvWarps];
    // what a cluster's CTAs write into each other
    unsigned lo[8], hi[8], prot[8], sum[8], bin, before, ties[8], holes[8], movers[8];
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
// rows, whose keys stay in shared memory (STAGED) or, above 40960 rows a CTA,
// in the workspace.  The key of the last row that stays is found by rounds of
// a histogram of 2048 equal steps over the range that is left of the keys
// (first that of the line's own keys, so weights of one magnitude still
// spread): three rounds at most.  Then rows are numbered in order, a
// neighbourhood per thread: who stays (keys above the threshold, the first
// rows at it), the places below the budget that become free, the rows beyond
// it that stay; the i-th of these will move into the i-th place.
// (Counting seven thresholds at once for eleven rounds took 17000 cycles of a
// line of 2176 rows, scans tile by tile as many.)
template <bool STAGED>
__global__ void __launch_bounds__(kEvThreads) k_evict_select(PagedEvictArgs a, int C) {
    extern __shared__ uint32_t staged[];
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
    auto total = [&](const unsigned *v) {
        unsigned t = 0;
        for (int q = 0; q < C; q++) t += v[q];
        return t;
    };
    if (C > 1) cl_arrive_relaxed();   // the others have started: waited for before the first store to them
    pdl_wait();
    const int n = paged_len(kv, b, tid == 0 && j == 0 && rank == 0), np = ld_now(a.next_pos + b);
    const int left = min(n, a.budget);
    const long long line = static_cast<long long>(line_no) * a.stride;
    const float *acc = a.acc + line;
    const int32_t *pos = a.pos + line;
    if (j == 0 && tid == 0 && rank == 0) a.lens_out[b] = left;
    const int slice = (n + C - 1) / C, first = min(n, rank * slice), len = min(n, first + slice) - first;
    uint32_t *keys = STAGED ? staged : a.keys + (static_cast<long long>(line_no) * kv.max_pages << kv.page_shift) + first;
    if (C > 1) cl_wait();
    if (n <= a.budget) {   // all stay (every CTA of the cluster comes here)
        for (int r = first + tid; r < first + len; r += kEvThreads) {
            a.acc_out[line + r] = acc[r];
            a.pos_out[line + r] = pos[r];
        }
        if (tid == 0 && rank == 0) a.moves[line_no] = 0;
        return;
    }
    // ---------------- keys, their range, the protected rows
    unsigned k_lo = 0xFFFFFFFFu, k_hi = 0, prot = 0;
#pragma unroll 4
    for (int i = tid; i < len; i += kEvThreads) {
        const uint32_t k = evict_key(acc[first + i], pos[first + i], np, a.n_recent, a.n_sink);
        keys[i] = k;
        if (k == kProtected) {
            prot++;
        } else {
            k_lo = min(k_lo, k);
            k_hi = max(k_hi, k);
        }
    }
    k_lo = __reduce_min_sync(0xffffffffu, k_lo);
    k_hi = __reduce_max_sync(0xffffffffu, k_hi);
    prot = __reduce_add_sync(0xffffffffu, prot);
    if (lane == 0) {
        sh.red[0][warp] = k_lo;
        sh.red[1][warp] = k_hi;
        sh.red[2][warp] = prot;
    }
    __syncthreads();
    if (warp == 0) {
        k_lo = __reduce_min_sync(0xffffffffu, lane < kEvWarps ? sh.red[0][lane] : 0xFFFFFFFFu);
        k_hi = __reduce_max_sync(0xffffffffu, lane < kEvWarps ? sh.red[1][lane] : 0u);
        prot = __reduce_add_sync(0xffffffffu, lane < kEvWarps ? sh.red[2][lane] : 0u);
        if (lane < C) {
            tell(&sh.lo[rank], k_lo, lane);
            tell(&sh.hi[rank], k_hi, lane);
            tell(&sh.prot[rank], prot, lane);
        }
    }
    all_sync();
    for (int q = 0; q < C; q++) {
        k_lo = q ? min(k_lo, sh.lo[q]) : sh.lo[0];
        k_hi = q ? max(k_hi, sh.hi[q]) : sh.hi[0];
    }
    prot = total(sh.prot);
    // ---------------- threshold: `ties` of the rows at thr stay, and all above it
    uint32_t thr = kProtected;
    unsigned ties = static_cast<unsigned>(left);
    if (prot < static_cast<unsigned>(left)) {
        unsigned need = static_cast<unsigned>(left) - prot;       // of the keys in [k_lo, k_hi], the largest
        while (k_hi > k_lo) {
            const int shift = max(0, 21 - __clz(k_hi - k_lo));    // (range >> shift) < 2048
#pragma unroll
            for (int i = 0; i < kEvBins / 4 / kEvThreads; i++)
                reinterpret_cast<uint4 *>(sh.hist)[tid + i * kEvThreads] = make_uint4(0, 0, 0, 0);
            __syncthreads();
#pragma unroll 4
            for (int i = tid; i < len; i += kEvThreads) {
                const uint32_t k = keys[i];
                if (k >= k_lo && k <= k_hi) atomicAdd(&sh.hist[(k_hi - k) >> shift], 1u);   // step 0: the largest
            }
            all_sync();
            // the CTA's share of the steps, added up over the cluster, scanned from the largest down
            const int share = kEvBins / C, per = (share + kEvThreads - 1) / kEvThreads, s0 = rank * share + tid * per;
            unsigned c[kEvShare], mine = 0;
#pragma unroll
            for (int i = 0; i < kEvShare; i++) {
                c[i] = 0;
                if (i < per && tid * per + i < share) {
                    if (C == 1) {
                        c[i] = sh.hist[s0 + i];
                    } else {
                        unsigned v[8];
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            v[q] = 0;
                            if (q < C)
                                asm volatile("ld.shared::cluster.u32 %0, [%1];"
                                             : "=r"(v[q])
                                             : "r"(cl_map(smem_addr(&sh.hist[s0 + i]), q))
                                             : "memory");
                        }
#pragma unroll
                        for (int q = 0; q < 8; q++) c[i] += v[q];
                    }
                }
                mine += c[i];
            }
            unsigned tot, before = cta_scan(mine, sh.scan, tot);
            if (C > 1) {
                if (tid < C) tell(&sh.sum[rank], tot, tid);
                all_sync();
                for (int q = 0; q < rank; q++) before += sh.sum[q];
            }
#pragma unroll
            for (int i = 0; i < kEvShare; i++) {
                if (before < need && need <= before + c[i])
                    for (int q = 0; q < C; q++) {
                        tell(&sh.bin, s0 + i, q);
                        tell(&sh.before, before, q);
                    }
                before += c[i];
            }
            all_sync();
            need -= sh.before;
            const uint32_t top = k_hi - (sh.bin << shift), width = (1u << shift) - 1;
            k_lo = top - k_lo > width ? top - width : k_lo;
            k_hi = top;
            __syncthreads();   // (bin and before are read before the next round writes them)
        }
        thr = k_lo;
        ties = need;
    }
    // ---------------- numbering, in row order: a thread's neighbouring rows (an odd number: no bank is met twice)
    const int per = ((len + kEvThreads - 1) / kEvThreads) | 1, i0 = min(len, tid * per), i1 = min(len, i0 + per);
    unsigned n_ties = 0, tot;
    for (int i = i0; i < i1; i++) n_ties += keys[i] == thr;
    unsigned tie = cta_scan(n_ties, sh.scan, tot);
    if (tid < C) tell(&sh.ties[rank], tot, tid);
    all_sync();
    for (int q = 0; q < rank; q++) tie += sh.ties[q];
    unsigned n_holes = 0, n_movers = 0;
    for (int i = i0; i < i1; i++) {
        const uint32_t k = keys[i];
        const bool stay = k > thr || (k == thr && tie < ties);
        tie += k == thr;
        keys[i] = stay;
        n_holes += !stay && first + i < left;
        n_movers += stay && first + i >= left;
    }
    unsigned hole = cta_scan(n_holes, sh.scan, tot);
    if (tid < C) tell(&sh.holes[rank], tot, tid);
    unsigned mover = cta_scan(n_movers, sh.scan, tot);
    if (tid < C) tell(&sh.movers[rank], tot, tid);
    all_sync();
    for (int q = 0; q < rank; q++) {
        hole += sh.holes[q];
        mover += sh.movers[q];
    }
    int32_t *from = a.src + static_cast<long long>(line_no) * a.budget, *to = a.places + static_cast<long long>(line_no) * a.budget;
    for (int i = i0; i < i1; i++) {
        if (!keys[i] && first + i < left) to[hole++] = first + i;
        if (keys[i] && first + i >= left) from[mover++] = first + i;
    }
    if (tid == 0 && rank == 0) a.moves[line_no] = static_cast<int32_t>(total(sh.movers));
    // rows that stay where they are
#pragma unroll 4
    for (int i = tid; i < min(len, left - first); i += kEvThreads)
        if (keys[i]) {
            a.acc_out[line + first + i] = acc[first + i];
            a.pos_out[line + first + i] = pos[first + i];
        }
    if (C > 1) all_sync();   // no CTA leaves while another reads its counts
}

// Warp = four moves of a line: weight, position, and K and V by 16-byte
// pieces, all four rows' loads in flight.  Sources lie at or beyond the
// budget, places below it, so no row is both.
__global__ void __launch_bounds__(256) k_evict_move(PagedEvictArgs a, int blocks, int row_bytes) {
    pdl_trigger();
    const PagedKv &kv = a.kv;
    const int line_no = blockIdx.x / blocks, b = line_no / kv.n_kv, j = line_no - b * kv.n_kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long line = static_cast<long long>(line_no) * a.stride;
    const int32_t *from_l = a.src + static_cast<long long>(line_no) * a.budget;
    const int32_t *to_l = a.places + static_cast<long long>(line_no) * a.budget;
    const int pieces = row_bytes / 16, size = row_bytes / kv.hd;
    pdl_wait();
    const int moves = ld_cg(a.moves + line_no);
    for (int i0 = ((blockIdx.x - line_no * blocks) * 8 + warp) * 4; i0 < moves; i0 += blocks * 32) {
        // lanes 0-3: the four sources, 4-7: their places; each looks its page up
        int r = 0;
        long long off = -1;
        if (lane < 8 && i0 + (lane & 3) < moves) {
            r = ld_cg((lane < 4 ? from_l : to_l) + i0 + (lane & 3));
            off = paged_off(kv, b, j, r);
            if (off < 0) atomicExch(kv.err, kErrBadPos);
        }
        const int place = __shfl_down_sync(0xffffffffu, r, 4);
        if (lane < 4 && i0 + lane < moves) {
            a.acc_out[line + place] = a.acc[line + r];
            a.pos_out[line + place] = a.pos[line + r];
        }
        long long from[4], to[4];
#pragma unroll
        for (int z = 0; z < 4; z++) {
            from[z] = __shfl_sync(0xffffffffu, off, z);
            to[z] = __shfl_sync(0xffffffffu, off, 4 + z);
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

// CTAs of a line: 4096 rows each, eight at most
static int evict_ctas(long long rows) {
    int C = 1;
    while (C < 8 && rows > 4096ll * C) C <<= 1;
    return C;
}
bool evict_staged(long long rows) { return (rows + evict_ctas(rows) - 1) / evict_ctas(rows) <= kEvSlice; }

cudaError_t launch_paged_evict(const PagedEvictArgs &a, int sms, cudaStream_t st) {
    const long long rows = static_cast<long long>(a.kv.max_pages) << a.kv.page_shift;
    const int C = evict_ctas(rows), lines = a.kv.n_seqs * a.kv.n_kv;
    const bool staged = evict_staged(rows);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(lines) * C);
    cfg.blockDim = dim3(kEvThreads);
    cfg.dynamicSmemBytes = staged ? static_cast<size_t>((rows + C - 1) / C) * 4 : 0;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = C > 1 ? 2 : 1;
    cudaError_t e = cudaSuccess;
    if (staged) e = allow_smem<k_evict_select<true>>(kEvSlice * 4);
    if (e == cudaSuccess)
        e = staged ? cudaLaunchKernelEx(&cfg, k_evict_select<true>, a, C) : cudaLaunchKernelEx(&cfg, k_evict_select<false>, a, C);
    if (e != cudaSuccess) return e;
    // four moves a warp, at most eight CTAs per SM in all
    const int blocks = std::max(1, std::min((a.budget + 31) / 32, 8 * sms / lines));
    return launch_pdl(k_evict_move, dim3(static_cast<unsigned>(lines) * blocks), dim3(256), 0, st, a, blocks,
                      a.kv.hd * (a.kv.dtype == STYX_F32 ? 4 : 2));
}

}  // namespace styx
