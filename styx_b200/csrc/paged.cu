// paged.cu -- rows into and out of a paged KV cache (include/styx_serve.h):
//
//   k_paged_append   per-head RMSNorm, RoPE and the rounded K / V rows
//   k_evict_select   the rows that stay, and the moves that close the gaps
//   k_evict_move     K, V, weight and position of the rows that move
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "cluster.cuh"
#include "paged.cuh"

namespace styx {
namespace {

// ------------------------------------------------------------ append
// A warp takes a token's rows (q heads, k heads, v heads), or a share of them:
// LPR lanes per row, lane l of them the pairs (i, i + d/2) of i = 4 l ... + 3,
// kAppRows x 32 / LPR rows at a time, all loads first.  The token's place and
// its cosines and sines, in the lane's registers for all its rows, are found
// while the first loads are on their way; nothing is shared between warps.
// The angle in turns, pos * base^(-2i/d) / 2 pi, is held in 64 bits and
// reduced to a fraction of a turn before it is rounded to f32, so its error
// does not grow with the position.
// Bound by HBM on prompts (8191 tokens of 32 q and 2 x 4 k / v heads of 128:
// 319 MB in 57 us, 5.6 TB/s; two rows at a time and 32 warps per SM: 65 us
// with four rows, whose registers spill at that many warps, 61 with four rows
// and 20 warps), by the latency of position, page and rows on a step of 64
// tokens (3.6 us).
constexpr int kAppThreads = 128, kAppRows = 2;

template <class T>
__device__ __forceinline__ void store4(T *p, const float (&v)[4]) {
    T u[4] = {from_f<T>(v[0]), from_f<T>(v[1]), from_f<T>(v[2]), from_f<T>(v[3])};
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(u);
    else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(u);
}

// VEC: d is a multiple of 8 and every row of the inputs is 16-byte aligned;
// else loads and stores are by element.  splits: warps per token, share rows
// each.
template <class T, int LPR, bool VEC>
__global__ void __launch_bounds__(kAppThreads, 8) k_paged_append(PagedAppendArgs a, int splits, int share) {
    pdl_trigger();
    constexpr int RPW = 32 / LPR;
    const PagedKv &kv = a.kv;
    const int hd = kv.hd, half = hd >> 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i0 = lane % LPR * 4, sub = lane / LPR, rows = a.n_heads + 2 * kv.n_kv;
    double turn[4];
    turn[0] = exp2(a.log2_base * i0) * 0.15915494309189535;   // 1 / 2 pi
#pragma unroll
    for (int e = 1; e < 4; e++) turn[e] = turn[e - 1] * a.step;
    bool in[4];
#pragma unroll
    for (int e = 0; e < 4; e++) in[e] = VEC ? i0 < half : i0 + e < half;
    pdl_wait();
    float wq[2][4], wk[2][4];
#pragma unroll
    for (int y = 0; y < 2; y++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            wq[y][e] = a.q_norm && in[e] ? ld_now(a.q_norm + y * half + i0 + e) : 1.f;
            wk[y][e] = a.k_norm && in[e] ? ld_now(a.k_norm + y * half + i0 + e) : 1.f;
        }
    const unsigned units = static_cast<unsigned>(a.n_tokens) * splits;
    for (unsigned u = blockIdx.x * (kAppThreads / 32) + warp; u < units; u += gridDim.x * (kAppThreads / 32)) {
        const int t = u / splits, h_begin = (u - t * splits) * share, h_end = min(rows, h_begin + share);
        float x[kAppRows][4], y[kAppRows][4];
        auto load = [&](int h0) {
#pragma unroll
            for (int j = 0; j < kAppRows; j++) {
                const int h = h0 + j * RPW + sub;
#pragma unroll
                for (int e = 0; e < 4; e++) x[j][e] = y[j][e] = 0.f;
                if (h < h_end && in[0]) {
                    const int hk = h - a.n_heads;
                    const float *src = hk < 0         ? a.q + t * a.q_stride + static_cast<long long>(h) * hd
                                       : hk < kv.n_kv ? a.k + t * a.k_stride + static_cast<long long>(hk) * hd
                                                      : a.v + t * a.v_stride + static_cast<long long>(hk - kv.n_kv) * hd;
                    if constexpr (VEC) {
                        *reinterpret_cast<float4 *>(x[j]) = *reinterpret_cast<const float4 *>(src + i0);
                        *reinterpret_cast<float4 *>(y[j]) = *reinterpret_cast<const float4 *>(src + half + i0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (in[e]) {
                                x[j][e] = src[i0 + e];
                                y[j][e] = src[half + i0 + e];
                            }
                    }
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
            const double f = pos * turn[e];
            sincospif(static_cast<float>(2.0 * (f - rint(f))), &s[e], &c[e]);
        }
        for (int h0 = h_begin;;) {
#pragma unroll
            for (int j = 0; j < kAppRows; j++) {
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
                    p[e] = is_v ? x[j][e] : x[j][e] * c[e] - y[j][e] * s[e];
                    q[e] = is_v ? y[j][e] : x[j][e] * s[e] + y[j][e] * c[e];
                    if (r < 0) p[e] = q[e] = 0.f;          // padding, or an empty slot
                }
                if (h >= h_end || !in[0]) continue;
                auto put = [&](auto *o) {
                    if constexpr (VEC) {
                        store4(o + i0, p);
                        store4(o + half + i0, q);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (in[e]) {
                                o[i0 + e] = from_f<std::remove_pointer_t<decltype(o)>>(p[e]);
                                o[half + i0 + e] = from_f<std::remove_pointer_t<decltype(o)>>(q[e]);
                            }
                    }
                };
                if (is_q) put(a.q_out + (static_cast<long long>(t) * a.n_heads + h) * hd);
                else if (row_ok)
                    put(static_cast<T *>(is_v ? kv.v : kv.k) + off +
                        (static_cast<long long>(is_v ? hk - kv.n_kv : hk) << kv.page_shift) * hd);
            }
            h0 += kAppRows * RPW;
            if (h0 >= h_end) break;
            load(h0);
        }
    }
}

template <class T>
cudaError_t append_t(const PagedAppendArgs &a, bool vec, int lpr, dim3 grid, int splits, int share, cudaStream_t st) {
    auto go = [&](auto *kern) { return launch_pdl(kern, grid, dim3(kAppThreads), 0, st, a, splits, share); };
    if (lpr == 8) return vec ? go(k_paged_append<T, 8, true>) : go(k_paged_append<T, 8, false>);
    if (lpr == 16) return vec ? go(k_paged_append<T, 16, true>) : go(k_paged_append<T, 16, false>);
    return vec ? go(k_paged_append<T, 32, true>) : go(k_paged_append<T, 32, false>);
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
    unsigned lo[8], hi[8], prot[8], sum[8], bin, before, in, ties[8], holes[8], movers[8];
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
// line of 2176 rows, scans tile by tile as many; counting 16 steps at once in
// registers made the whole call 28 us instead of 22, since weights spread over
// many exponents and then take eight rounds.)
// Bound by the chain of exchanges, not by bytes: with the moves, 18.3 us from
// 32768 rows to 4096 (one sequence, 4 kv heads; 2.5 us at HBM's rate: keys 4,
// threshold 7, numbering 1.5, places 2), 19.2 us for 32 sequences from 2176 to
// 2048 (3.1; keys 2.5, threshold 4, numbering 1, moves 5, two launches), in a
// graph over one state; 21 and 20 as called over several.
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
        if (first + i < left) {   // (a row that leaves: overwritten by the one that moves to its place)
            a.acc_out[line + first + i] = acc[first + i];
            a.pos_out[line + first + i] = pos[first + i];
        }
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
        unsigned in = static_cast<unsigned>(n) - prot;            // that many there are
        while (k_hi > k_lo && in > need) {
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
                        tell(&sh.in, c[i], q);
                    }
                before += c[i];
            }
            all_sync();
            need -= sh.before;
            in = sh.in;
            const uint32_t top = k_hi - (sh.bin << shift), width = (1u << shift) - 1;
            k_lo = top - k_lo > width ? top - width : k_lo;
            k_hi = top;
            __syncthreads();   // (bin and before are read before the next round writes them)
        }
        thr = in > need ? k_lo : k_lo - 1;   // (all of the range stay; no key is 0)
        ties = in > need ? need : 0;
    }
    // ---------------- numbering, in row order: a thread's neighbouring rows (an odd number: no bank is met twice)
    const int per = ((len + kEvThreads - 1) / kEvThreads) | 1, i0 = min(len, tid * per), i1 = min(len, i0 + per);
    unsigned tie = 0, tot;
    if (ties > 0) {   // (the same for all CTAs of the line)
        unsigned n_ties = 0;
        for (int i = i0; i < i1; i++) n_ties += keys[i] == thr;
        tie = cta_scan(n_ties, sh.scan, tot);
        if (tid < C) tell(&sh.ties[rank], tot, tid);
        all_sync();
        for (int q = 0; q < rank; q++) tie += sh.ties[q];
    }
    unsigned n_holes = 0, n_movers = 0;
    for (int i = i0; i < i1; i++) {
        const uint32_t k = keys[i];
        const bool stay = k > thr || (k == thr && tie < ties);
        tie += k == thr;
        keys[i] = stay;
        n_holes += !stay && first + i < left;
        n_movers += stay && first + i >= left;
    }
    unsigned hole, mover;
    if constexpr (STAGED) {   // (fewer than 2^16 of each in a CTA)
        const unsigned both = cta_scan(n_movers << 16 | n_holes, sh.scan, tot);
        hole = both & 0xFFFFu;
        mover = both >> 16;
        if (tid < C) {
            tell(&sh.holes[rank], tot & 0xFFFFu, tid);
            tell(&sh.movers[rank], tot >> 16, tid);
        }
    } else {
        hole = cta_scan(n_holes, sh.scan, tot);
        if (tid < C) tell(&sh.holes[rank], tot, tid);
        mover = cta_scan(n_movers, sh.scan, tot);
        if (tid < C) tell(&sh.movers[rank], tot, tid);
    }
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
    const int rows = a.n_heads + 2 * a.kv.n_kv, hd = a.kv.hd, lpr = hd <= 64 ? 8 : hd <= 128 ? 16 : 32;
    const int batch = kAppRows * (32 / lpr), batches = (rows + batch - 1) / batch;
    // warps per token: one where that fills the SMs (24 warps each), else as many as there are batches of rows
    // (8191 tokens of 32 + 2 x 4 rows: 61 us with one warp each, 69 with three, 72 with five, at four rows at a time;
    // 64 tokens: 4.1 us with five)
    const long long want = (24ll * sms + a.n_tokens - 1) / a.n_tokens;
    const int share = (batches + static_cast<int>(std::min<long long>(batches, want)) - 1) /
                      static_cast<int>(std::min<long long>(batches, want)) * batch;
    const int splits = (rows + share - 1) / share;
    const long long ctas = (static_cast<long long>(a.n_tokens) * splits + kAppThreads / 32 - 1) / (kAppThreads / 32);
    const dim3 grid(static_cast<unsigned>(std::min<long long>(ctas, 32ll * sms)));
    auto al16 = [](const void *p, long long s) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s % 4 == 0; };
    const bool vec = hd % 8 == 0 && al16(a.q, a.q_stride) && al16(a.k, a.k_stride) && al16(a.v, a.v_stride);
    return a.kv.dtype == STYX_F16    ? append_t<__half>(a, vec, lpr, grid, splits, share, st)
           : a.kv.dtype == STYX_BF16 ? append_t<__nv_bfloat16>(a, vec, lpr, grid, splits, share, st)
                                     : append_t<float>(a, vec, lpr, grid, splits, share, st);
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
