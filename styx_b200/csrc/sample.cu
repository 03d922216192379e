// sample.cu -- temperature, top-k, top-p, min-p and the draw
// (styx_sample, include/styx_serve.h).
//
// The kept tokens are a prefix of the order (larger logit, lower index), so
// they are described by one threshold: all tokens whose key is above it and
// the first `ties` of those at it.  Weights are whole numbers (2^-40 of the
// largest one's), so every sum is exact whatever its order.
//
// k_sample_cluster (n_vocab <= 262144): a cluster of eight CTAs per row holds
// the row in shared memory, so the logits are read once.
//   top-k up to 120: the k-th largest of the cluster's 128 warps' maxima is a
//     bound that the k-th largest logit reaches; the tokens at or above it
//     (22 on average for k = 20, 355 for 120, where large ones are spread
//     evenly) go to the cluster's first CTA, which sorts them and does the rest.
//   else, with top-k or top-p: one histogram over 2048 equal steps of log
//     weight (tokens below e^-28 have weight 0 and take no part in anything),
//     of counts or of weights, shows the step in which the threshold lies;
//     each CTA adds up an eighth of it (all of it in every CTA was 190 KB
//     over distributed shared memory, 12000 cycles).  Where the tokens down to
//     there are at most 2048 they go to the first CTA as above; else only that
//     step's tokens go there and the threshold comes back.  Top-p after such
//     a top-k is a second histogram, of the tokens kept.  Only more than 2048
//     tokens in one step (a flat row, or very many tokens at a high temperature)
//     are resolved by bisection of the key, up to 32 passes over the slices with
//     a cluster barrier each: a flat row of 151936 with top-p 0.5 251 us, 64 of
//     them 791; 200000 tokens of spread 1 at temperature 3, top-p 0.5, 371 us.
//   the draw, where it is not the first CTA's: sums of the kept weights per
//     warp, each over a stretch of indexes of its own, then inside one warp.
// Measured (B200, vocabulary 151936): one row with top-k 20 and top-p 0.95 in
// 7.5 us, the maximum alone 6.5, without filters 12, with top-p over all of it
// 34 to 36 (the histogram 8 of them); 64 rows of mixed settings 52.5 us (39 MB:
// 6 at HBM's rate), of which the rows with a histogram, begun first, take 38;
// in the order given 61.
// (The row in registers, 1024 threads of 64, spilled; a conversion of the
// weights by F2I and sums per round of the CTA made the draw of an unfiltered
// row 18000 of 34000 cycles.)
//
// k_sample (larger vocabularies): one CTA per row, radix selection from L2, the
// row read up to twelve times.  300000 tokens: 1.0 ms unfiltered, 4.7 to 4.9
// greedy, with top-k or top-p; 64 rows 1.7 and 8.0 to 8.4 ms.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "cluster.cuh"
#include "kernels.h"

namespace styx {
namespace {

constexpr int kThreads = 1024;
using u64 = unsigned long long;

__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }   // NaN: -inf; -0: +0
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// floor(of * total / 2^24) for of <= 2^24
__device__ __forceinline__ u64 part_of(u64 of, u64 total) {
    return (total >> 24) * of + (((total & 0xFFFFFFu) * of) >> 24);
}

// floor(w 2^40) for 0 <= w <= 1, by its bits (a conversion to 64 bits costs
// several times the shift)
__device__ __forceinline__ u64 whole_of(float w) {
    const uint32_t b = __float_as_uint(w), f = (b & 0x7FFFFFu) | 0x800000u;
    return (static_cast<u64>(f) << 17) >> min(127u - (b >> 23), 63u);   // (below 2^-40, and 0: shifted out)
}

struct Row {
    const float *x;
    float m, inv_t;
    bool hot;
    // inv_t: infinite for the greedy pick, else finite and above 0, so that (v - m) inv_t is no NaN
    __device__ __forceinline__ float weight(float v) const { return v == m ? 1.f : expf((v - m) * inv_t); }
    __device__ __forceinline__ u64 whole(float v) const { return whole_of(weight(v)); }
};

template <class V>
__device__ __forceinline__ V block_sum(V v, V *red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// exclusive prefix over the block of (sum a); total in `tot`
template <class V>
__device__ __forceinline__ V block_prefix(V v, V *red, V &tot) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    V s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 31) red[w] = s;
    __syncthreads();
    V x = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
    }
    tot = __shfl_sync(0xffffffffu, x, 31);
    const V before = __shfl_sync(0xffffffffu, x, w ? w - 1 : 0);
    return (w ? before : V(0)) + s - v;
}

// Selection by radix, four digits of 8 bits from the top, over the keys at or
// above (thr0, the first ties0 of equals): finds the key at which the running
// sum of `measure` (1 or the weight) from the top first reaches `need`, and
// how many of the tokens at that key that takes.  `above`: the sum over the
// keys above it.
template <bool BY_WEIGHT>
__device__ void select(const Row &row, int n, u64 need, uint32_t thr0, u64 *hist, u64 *sh, uint32_t &thr, u64 &above) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    u64 sum = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const float v = clean(row.x[i]);
            const uint32_t k = key_of(v);
            if (k < thr0) continue;
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
                atomicAdd(&hist[(k >> shift) & 255], BY_WEIGHT ? row.whole(v) : 1ull);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255;
            for (; d > 0; d--) {
                if (sum + hist[d] >= need) break;
                sum += hist[d];
            }
            sh[0] = prefix | (static_cast<uint32_t>(d) << shift);
            sh[1] = sum;
        }
        __syncthreads();
        prefix = static_cast<uint32_t>(sh[0]);
        sum = sh[1];
    }
    thr = prefix;
    above = sum;
}

__global__ void __launch_bounds__(kThreads) k_sample(SampleArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ u64 red[32], hist[256], sh[2];
    __shared__ float redf[32];
    __shared__ int s_token;
    const int b = blockIdx.x, n = a.n_vocab, tid = threadIdx.x;
    Row row;
    row.x = a.logits + b * a.row_stride;
    const float t = a.temperature ? a.temperature[b] : 1.f;
    row.hot = t > 0.f;
    row.inv_t = row.hot ? fmaxf(1.0f / t, 0x1p-126f) : INFINITY;
    float m = -INFINITY;
    for (int i = tid; i < n; i += kThreads) m = fmaxf(m, clean(row.x[i]));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) redf[tid >> 5] = m;
    __syncthreads();
    m = redf[tid & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    row.m = m;
    if (!(m > -INFINITY)) {   // nothing to draw from
        if (tid == 0) {
            a.token[b] = -1;
            if (a.logprob) a.logprob[b] = -INFINITY;
        }
        return;
    }
    int k = a.top_k ? a.top_k[b] : 0;
    if (k <= 0 || k > n) k = n;
    if (!row.hot) k = 1;
    uint32_t thr = 0;      // kept: keys above thr, and the first `ties` at it
    u64 ties = ~0ull, total;
    // the weight of a key: any logit with it has the same
    auto weight_of_key = [&](uint32_t key) {
        const uint32_t bits = (key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key;
        return row.whole(__uint_as_float(bits));
    };
    if (k < n) {
        u64 above;
        select<false>(row, n, static_cast<u64>(k), 0, hist, sh, thr, above);
        ties = static_cast<u64>(k) - above;
    }
    u64 s = 0;
    for (int i = tid; i < n; i += kThreads) {
        const float v = clean(row.x[i]);
        const uint32_t key = key_of(v);
        if (key > thr || (ties == ~0ull && key == thr)) s += row.whole(v);
    }
    total = block_sum(s, red);
    if (ties != ~0ull) total += ties * weight_of_key(thr);
    const float p = a.top_p ? fminf(a.top_p[b], 1.f) : 1.f;
    const u64 p24 = p > 0.f ? static_cast<u64>(rintf(p * 0x1p24f)) : 0ull;
    if (p24 < (1ull << 24)) {
        const u64 need = max(part_of(p24, total), 1ull);
        uint32_t thr2;
        u64 above;
        select<true>(row, n, need, thr, hist, sh, thr2, above);
        const u64 w = weight_of_key(thr2);
        u64 c = w ? (need - above + w - 1) / w : ~0ull;   // the tokens at thr2 that the sum takes
        if (thr2 == thr) c = min(c, ties);
        thr = thr2;
        ties = c;
    }
    // min-p, the draw: two passes in index order
    const float mp = a.min_p ? fminf(a.min_p[b], 1.f) : 0.f;   // the maximum always stays
    u64 sum = 0, seen = 0;
    for (int pass = 0; pass < 2; pass++) {
        u64 target = 0;
        if (pass == 1) {
            const float u = fminf(fmaxf(a.u[b], 0.f), 0x1.fffffep-1f);
            target = part_of(static_cast<u64>(u * 0x1p24f), sum);
            total = sum;
            sum = 0;
            seen = 0;
            if (tid == 0) s_token = -1;
            __syncthreads();
        }
        for (int base = 0; base < n; base += kThreads) {
            const int i = base + tid;
            const float v = i < n ? clean(row.x[i]) : -INFINITY;
            const uint32_t key = key_of(v);
            u64 tot;
            const u64 at = seen + block_prefix(static_cast<u64>(i < n && key == thr), red, tot);
            seen += tot;
            const bool in = i < n && (key > thr || (key == thr && at < ties)) && row.weight(v) >= mp;
            const u64 w = in ? row.whole(v) : 0ull;
            const u64 before = sum + block_prefix(w, red, tot);
            sum += tot;
            if (pass == 1 && before <= target && target < before + w) s_token = i;
        }
        __syncthreads();
    }
    if (tid == 0) {
        const int i = s_token;
        a.token[b] = i;
        if (a.logprob) {
            float lp = -INFINITY;
            if (i >= 0) {
                const float v = clean(row.x[i]);
                lp = (v == m ? 0.f : (v - m) * row.inv_t) - logf(static_cast<float>(total) * 0x1p-40f);
            }
            a.logprob[b] = lp;
        }
    }
}

// ------------------------------------------------------------ one cluster per row
constexpr int kC = 8;                       // CTAs of a row
constexpr int kNT = 512, kNW = kNT / 32;    // threads and warps of a CTA
constexpr int kBins = 4 * kNT, kCap = 4 * kNT, kShare = kBins / kC;
constexpr float kBinScale = kBins / 28.f;
constexpr int kSlice = 32768;               // logits of a CTA at most
constexpr int kTopK = 120;                  // top-k by the warps' maxima (128 of them)

struct CtaShared {
    union {
        __align__(16) unsigned hist[3][kBins];            // counts, or the low and high words of the weights' sums (0, 1)
        u64 cand[kCap];                     // (inverted key << 32) | index: ascending = the order of the tokens
    };
    u64 red[32], ent[2][kNW + 1];
    uint64_t bar;
    float bound;
    unsigned n_mine;
    // what the cluster's CTAs write into each other
    __align__(16) float top[kC * kNW];
    u64 sum[2][kC], before, ties;
    unsigned cnt[2][kC], n_of[kC], step, thr;
    int n_of_warp[kNW], row;                // the order of the rows
};
static_assert(offsetof(CtaShared, hist) % 16 == 0 && offsetof(CtaShared, top) % 16 == 0, "read by 16 bytes");

__device__ __forceinline__ void cluster_sync() {
    cl_arrive();
    cl_wait();
}
__device__ __forceinline__ void st_u32(uint32_t addr, unsigned v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_u64(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned ld_u32(uint32_t addr) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v) {   // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}
// exclusive prefix and total over the CTA's kNT threads; total alone
__device__ __forceinline__ u64 cta_prefix(u64 v, u64 *red, u64 &tot) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const u64 s = warp_scan64(v);
    __syncthreads();
    if (lane == 31) red[w] = s;
    __syncthreads();
    const u64 x = warp_scan64(lane < kNW ? red[lane] : 0ull);
    tot = __shfl_sync(0xffffffffu, x, 31);
    const u64 before = __shfl_sync(0xffffffffu, x, w ? w - 1 : 0);
    return (w ? before : 0ull) + s - v;
}
__device__ __forceinline__ u64 cta_sum(u64 v, u64 *red) {
    const int lane = threadIdx.x & 31;
    v = warp_sum64(v);
    __syncthreads();
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum64(lane < kNW ? red[lane] : 0ull);
}
__device__ __forceinline__ float logit_of_key(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// E values per thread, neighbours: strides below E in registers, below 32 E by
// shuffles, the rest through buf
template <int E>
__device__ __forceinline__ void cta_sort_regs(u64 *buf) {
    const int t = threadIdx.x;
    u64 v[E];
#pragma unroll
    for (int i = 0; i < E; i++) v[i] = buf[E * t + i];
    for (int size = 2; size <= E * kNT; size <<= 1) {
        for (int stride = size >> 1; stride >= 32 * E; stride >>= 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; i++) buf[E * t + i] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int at = E * t + i;
                const u64 w = buf[at ^ stride];
                v[i] = ((at & stride) == 0) == ((at & size) == 0) ? min(v[i], w) : max(v[i], w);
            }
        }
        for (int stride = min(size >> 1, 16 * E); stride >= E; stride >>= 1)
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int at = E * t + i;
                const u64 w = __shfl_xor_sync(0xffffffffu, v[i], stride / E);
                v[i] = ((at & stride) == 0) == ((at & size) == 0) ? min(v[i], w) : max(v[i], w);
            }
#pragma unroll
        for (int stride = E / 2; stride; stride >>= 1)
            if (stride < size)
#pragma unroll
                for (int i = 0; i < E; i++)
                    if ((i & stride) == 0) {
                        const u64 x = v[i], y = v[i + stride];
                        const bool up = ((E * t + i) & size) == 0;
                        v[i] = up ? min(x, y) : max(x, y);
                        v[i + stride] = up ? max(x, y) : min(x, y);
                    }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; i++) buf[E * t + i] = v[i];
    __syncthreads();
}

// buf[0, n) sorted ascending (n a power of two, 32 or more): bitonic; up to one
// value per thread, strides below a warp by shuffles
__device__ __forceinline__ void cta_sort(u64 *buf, int n) {
    const int t = threadIdx.x;
    __syncthreads();
    if (n > kNT) {
        if (n == 2 * kNT) cta_sort_regs<2>(buf);
        else cta_sort_regs<4>(buf);
        return;
    }
    u64 v = t < n ? buf[t] : ~0ull;
    for (int size = 2; size <= n; size <<= 1) {
        const bool up = (t & size) == 0;
        for (int stride = size >> 1; stride >= 32; stride >>= 1) {
            __syncthreads();
            if (t < n) buf[t] = v;
            __syncthreads();
            const u64 w = t < n ? buf[t ^ stride] : ~0ull;
            v = ((t & stride) == 0) == up ? min(v, w) : max(v, w);
        }
        for (int stride = min(size >> 1, 16); stride; stride >>= 1) {
            const u64 w = __shfl_xor_sync(0xffffffffu, v, stride);
            v = ((t & stride) == 0) == up ? min(v, w) : max(v, w);
        }
    }
    __syncthreads();
    if (t < n) buf[t] = v;
    __syncthreads();
}

// slice: logits of a CTA, kNW * region of them, a warp's stretch each (region
// a multiple of 128).  bulk: the slices start on 16 bytes, and one bulk copy
// brings a CTA's.
// by_weight: clusters take the rows that need a histogram first, so that none
// of these is begun when the others are done (rows more than fit the SMs at
// once, settings for no more than a CTA's threads)
__global__ void __launch_bounds__(kNT, 2) k_sample_cluster(SampleArgs a, int region, bool bulk, bool by_weight) {
    extern __shared__ __align__(128) float xs[];
    __shared__ __align__(16) CtaShared sh;
    pdl_trigger();
    cl_arrive_relaxed();                          // the others have started: waited for before the first store to them
    const uint32_t rank = cluster_ctarank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = a.n_vocab;
    int b = blockIdx.x / kC;
    const int slice = kNW * region, lo = static_cast<int>(rank) * slice, len = max(0, min(n - lo, slice));
    const int first = warp * region;              // the warp's stretch of the slice
    auto peer = [&](const void *p, uint32_t r) { return cl_map(smem_addr(p), r); };
    const uint4 z4 = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        sh.n_mine = 0;
        mbar_init(&sh.bar, 1);
        fence_mbar_init();
    }
    pdl_wait();
    if (by_weight) {
        bool heavy = false;
        if (tid < a.n_rows) {
            const int k = a.top_k ? a.top_k[tid] : 0;
            const bool all = k <= 0 || k >= n;
            heavy = !(a.temperature && !(a.temperature[tid] > 0.f)) && (all ? a.top_p && a.top_p[tid] < 1.f : k > kTopK);
        }
        const unsigned votes = __ballot_sync(0xffffffffu, heavy);
        if (lane == 0) sh.n_of_warp[warp] = __popc(votes);
        __syncthreads();
        int before = __popc(votes & ((1u << lane) - 1)), all = 0;
        for (int w = 0; w < kNW; w++) {
            before += w < warp ? sh.n_of_warp[w] : 0;
            all += sh.n_of_warp[w];
        }
        if (tid < a.n_rows && (heavy ? before : all + tid - before) == b) sh.row = tid;
        __syncthreads();
        b = sh.row;
    }
    // ---------------- the slice, once; the warps' maxima
    const float *src = a.logits + b * a.row_stride + lo;
    const int whole4 = bulk ? len & ~3 : 0;
    if (tid == 0 && whole4) {
        mbar_arrive_expect_tx(&sh.bar, static_cast<uint32_t>(whole4) * 4);
        bulk_g2s(xs, src, static_cast<uint32_t>(whole4) * 4, &sh.bar);
    }
    const float t = a.temperature ? a.temperature[b] : 1.f, top_p = a.top_p ? a.top_p[b] : 1.f;
    const float min_p = a.min_p ? a.min_p[b] : 0.f, u = a.u[b];
    int k = a.top_k ? a.top_k[b] : 0;
    for (int i = whole4 + tid; i < slice; i += kNT) xs[i] = i < len ? src[i] : -INFINITY;
    __syncthreads();
    if (whole4) mbar_wait(&sh.bar, 0, a.err, kErrWaitFull);
    Row row;
    row.x = nullptr;
    row.hot = t > 0.f;
    // (an infinite temperature: no product with -inf may be NaN)
    row.inv_t = row.hot ? fmaxf(1.0f / t, 0x1p-126f) : INFINITY;
    const float p = fminf(top_p, 1.f), mp = fminf(min_p, 1.f);   // the maximum always stays
    const u64 p24 = p > 0.f ? static_cast<u64>(rintf(p * 0x1p24f)) : 0ull;
    const u64 u24 = static_cast<u64>(fminf(fmaxf(u, 0.f), 0x1.fffffep-1f) * 0x1p24f);
    float m = -INFINITY;
#pragma unroll 4
    for (int i = first + 4 * lane; i < first + region; i += 128) {
        const float4 v = *reinterpret_cast<const float4 *>(xs + i);
        const float4 c = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
        const uint4 d = make_uint4(__float_as_uint(v.x) ^ __float_as_uint(c.x), __float_as_uint(v.y) ^ __float_as_uint(c.y),
                                   __float_as_uint(v.z) ^ __float_as_uint(c.z), __float_as_uint(v.w) ^ __float_as_uint(c.w));
        if (d.x | d.y | d.z | d.w) *reinterpret_cast<float4 *>(xs + i) = c;
        m = fmaxf(m, fmaxf(fmaxf(c.x, c.y), fmaxf(c.z, c.w)));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    cl_wait();
    if (lane < kC) cl_st(peer(&sh.top[rank * kNW + warp], lane), m);
    cluster_sync();
    {
        const float4 v = reinterpret_cast<const float4 *>(sh.top)[lane];   // 128 maxima, four a lane
        m = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    row.m = m;
    if (!(m > -INFINITY)) {   // nothing to draw from
        if (rank == 0 && tid == 0) {
            a.token[b] = -1;
            if (a.logprob) a.logprob[b] = -INFINITY;
        }
        return;
    }
    if (!row.hot) k = 1;
    if (k <= 0 || k > n) k = n;
    const bool by_k = k < n, by_p = p24 < (1ull << 24);
    // all of the slice's logits, (place in the slice, logit)
    auto each = [&](auto f) {
#pragma unroll 2
        for (int i = first + 4 * lane; i < first + region; i += 128) {
            const float4 v = *reinterpret_cast<const float4 *>(xs + i);
            f(i, v.x);
            f(i + 1, v.y);
            f(i + 2, v.z);
            f(i + 3, v.w);
        }
    };
    auto finish = [&](int i, float v, u64 total) {   // by the thread that has the token
        a.token[b] = i;
        if (a.logprob)
            a.logprob[b] = (v == m ? 0.f : (v - m) * row.inv_t) - logf(static_cast<float>(total) * 0x1p-40f);
    };
    auto as_cand = [&](int i, float v) {
        return (static_cast<u64>(~key_of(v)) << 32) | static_cast<unsigned>(lo + i);
    };
    // the first CTA, with nc candidates (cand(i), any order) among which is all that is kept: sorted, top-k and top-p
    // keep the first ones, min-p too; then the draw in index order.  need_p: top-p's sum, where it is known.
    u64 *buf = reinterpret_cast<u64 *>(xs);       // (its own logits are no longer needed then)
    auto solve = [&](int nc, auto cand, bool p_known, u64 need_p) {
        if (nc <= 96) {
            // few: each candidate's thread counts and sums over the others
            u64 *wk = buf + 128, *wd = buf + 256;
            const u64 v = tid < nc ? cand(tid) : ~0ull;
            const uint32_t key = ~static_cast<uint32_t>(v >> 32);
            const float xv = logit_of_key(key);
            const u64 w = tid < nc ? row.whole(xv) : 0ull;
            __syncthreads();
            if (tid < nc) buf[tid] = v;
            __syncthreads();
            int place = 0;
            if (tid < nc) {
                for (int i = 0; i < nc; i++) place += buf[i] < v;
                wk[tid] = place < k ? w : 0ull;
            }
            __syncthreads();
            if (tid < nc) {
                bool kept = place < k && row.weight(xv) >= mp;
                if (by_p) {
                    u64 before = 0, tot = 0;
                    for (int i = 0; i < nc; i++) {
                        const u64 x = wk[i];
                        before += buf[i] < v ? x : 0ull;
                        tot += x;
                    }
                    kept = kept && before < (p_known ? need_p : max(part_of(p24, tot), 1ull));
                }
                wd[tid] = kept ? w : 0ull;
            }
            __syncthreads();
            if (tid < nc && wd[tid]) {
                u64 at = 0, tot = 0;
                for (int i = 0; i < nc; i++) {
                    const u64 x = wd[i];
                    at += static_cast<uint32_t>(buf[i]) < static_cast<uint32_t>(v) ? x : 0ull;
                    tot += x;
                }
                const u64 target = part_of(u24, tot);
                if (at <= target && target < at + wd[tid]) finish(static_cast<int>(static_cast<uint32_t>(v)), xv, tot);
            }
            return;
        }
        int n2 = 32;
        while (n2 < nc) n2 <<= 1;
        int per = max(1, n2 / kNT), i0 = tid * per;   // a thread's values, neighbours
        __syncthreads();
        for (int i = tid; i < n2; i += kNT) buf[i] = i < nc ? cand(i) : ~0ull;
        cta_sort(buf, n2);
        u64 before = 0, tot = 0;
        if (by_p) {
            u64 w = 0;
            for (int i = i0; i < i0 + per && i < min(nc, k); i++) w += row.whole(logit_of_key(~static_cast<uint32_t>(buf[i] >> 32)));
            before = cta_prefix(w, sh.red, tot);
        }
        const u64 need = !by_p ? ~0ull : p_known ? need_p : max(part_of(p24, tot), 1ull);
        unsigned n_kept = 0;
        for (int i = i0; i < i0 + per && i < n2; i++) {
            const u64 v = buf[i];
            const uint32_t key = ~static_cast<uint32_t>(v >> 32);
            const float xv = logit_of_key(key);
            const bool in = i < nc && i < k;
            const bool kept = in && before < need && row.weight(xv) >= mp;
            if (by_p && in) before += row.whole(xv);
            buf[i] = kept ? ((v & 0xFFFFFFFFull) << 32) | key : ~0ull;
            n_kept += kept;
        }
        // (the kept ones are the first of the order)
        n_kept = static_cast<unsigned>(cta_sum(n_kept, sh.red));
        n2 = 32;
        while (n2 < static_cast<int>(n_kept)) n2 <<= 1;
        per = max(1, n2 / kNT);
        i0 = tid * per;
        cta_sort(buf, n2);
        u64 w = 0;
        for (int i = i0; i < i0 + per && i < n2; i++)
            if (buf[i] != ~0ull) w += row.whole(logit_of_key(static_cast<uint32_t>(buf[i])));
        u64 at = cta_prefix(w, sh.red, tot);
        const u64 target = part_of(u24, tot);
        for (int i = i0; i < i0 + per && i < n2; i++) {
            const u64 z = buf[i];
            if (z == ~0ull) break;
            const float zx = logit_of_key(static_cast<uint32_t>(z));
            const u64 zw = row.whole(zx);
            if (at <= target && target < at + zw) finish(static_cast<int>(z >> 32), zx, tot);
            at += zw;
        }
    };
    uint32_t thr = 0;          // kept: keys above thr, and the first `ties` at it
    u64 ties = 0;
    if (by_k && k <= kTopK) {
        // the k-th largest of the 128 maxima: four threads each count a quarter of those before maximum t
        {
            const int t = tid >> 2, i0 = (tid & 3) * 4;
            const float mine = sh.top[t];
            int before = 0;
#pragma unroll
            for (int i = i0; i < kC * kNW; i += 16) {
                const float4 v = *reinterpret_cast<const float4 *>(&sh.top[i]);
                before += (v.x > mine || (v.x == mine && i < t)) + (v.y > mine || (v.y == mine && i + 1 < t)) +
                          (v.z > mine || (v.z == mine && i + 2 < t)) + (v.w > mine || (v.w == mine && i + 3 < t));
            }
            before += __shfl_xor_sync(0xffffffffu, before, 1);
            before += __shfl_xor_sync(0xffffffffu, before, 2);
            if (before == k - 1 && (tid & 3) == 0) sh.bound = mine;
        }
        __syncthreads();
        const float bound = sh.bound;
        constexpr unsigned kSeg = kCap / kC;       // the first CTA's places for each CTA's candidates
        if (bound > -INFINITY)
            each([&](int i, float v) {
                if (v >= bound) {
                    const unsigned at = atomicAdd(&sh.n_mine, 1u);
                    if (at < kSeg) st_u64(peer(&sh.cand[rank * kSeg + at], 0), as_cand(i, v));
                }
            });
        __syncthreads();
        if (tid < kC) st_u32(peer(&sh.n_of[rank], tid), bound > -INFINITY ? sh.n_mine : kSeg + 1);
        cluster_sync();
        int nc = 0;
        bool fits = true;
#pragma unroll
        for (int r = 0; r < kC; r++) {
            nc += sh.n_of[r];
            fits = fits && sh.n_of[r] <= kSeg;
        }
        if (fits) {
            if (rank == 0)
                solve(nc, [&](int i) {
                    int r = 0;
                    while (i >= static_cast<int>(sh.n_of[r])) i -= sh.n_of[r++];
                    return sh.cand[r * kSeg + i];
                }, false, 0);
            return;
        }
    }
    // the step of a token: kBins or more where the weight is 0
    const float bs = row.inv_t * kBinScale;
    auto step_of = [&](float v) { return v == m ? 0 : static_cast<int>(fminf((m - v) * bs, kBins)); };
    // Sum over the row's keys >= from of 1 or the weight; of the keys at floor_key only floor_ties count, none below it.
    auto measure = [&](uint32_t from, uint32_t floor_key, u64 floor_ties, bool weights, int slot) {
        u64 s = 0, eq = 0;
        each([&](int, float v) {
            const uint32_t key = key_of(v);
            if (key < from || key < floor_key || step_of(v) >= kBins) return;
            if (key == floor_key) eq++;
            else s += weights ? row.whole(v) : 1ull;
        });
        s = cta_sum(s, sh.red);
        eq = cta_sum(eq, sh.red);
        if (tid < kC) {
            st_u64(peer(&sh.sum[slot][rank], tid), s);
            st_u32(peer(&sh.cnt[slot][rank], tid), static_cast<unsigned>(eq));
        }
        cluster_sync();
        u64 all = 0, q = 0;
#pragma unroll
        for (int r = 0; r < kC; r++) {
            all += sh.sum[slot][r];
            q += sh.cnt[slot][r];
        }
        return all + min(q, floor_ties) * (weights ? row.whole(logit_of_key(floor_key)) : 1ull);
    };
    // the largest key whose sum reaches lim, and how many of the tokens at it that takes
    auto bisect = [&](u64 lim, bool weights, uint32_t floor_key, u64 floor_ties) {
        cluster_sync();   // every CTA has read the counts that it decided by: the first sum overwrites their slots
        uint32_t l = max(floor_key, 1u), h = key_of(m);   // measure(l) >= lim
        int slot = 0;
        while (l < h) {
            const uint32_t mid = l + (h - l) / 2 + 1;
            if (measure(mid, floor_key, floor_ties, weights, slot) >= lim) l = mid;
            else h = mid - 1;
            slot ^= 1;
        }
        const u64 above = measure(l + 1, l + 1, ~0ull, weights, slot);
        const u64 w = weights ? max(row.whole(logit_of_key(l)), 1ull) : 1ull;
        thr = l;
        ties = (lim - above + w - 1) / w;
        if (l == floor_key) ties = min(ties, floor_ties);
        cluster_sync();
    };
    // round 0: top-k by counts; round 1: top-p by weights, of what top-k has kept (keys above thr, `ties` at it)
    for (int round = by_k ? 0 : 1; round < (by_p ? 2 : 1); round++) {
        const bool weigh = round == 1;
        const uint32_t fk = thr;
        const u64 ft = ties, fw = fk ? row.whole(logit_of_key(fk)) : 0ull;
        cluster_sync();                                      // nothing of an earlier use of the histogram is in flight
#pragma unroll
        for (int i = 0; i < 3; i++) reinterpret_cast<uint4 *>(sh.hist[i])[tid] = z4;
        __syncthreads();
        const float x_floor = fk ? logit_of_key(fk) : -INFINITY;
        each([&](int, float v) {
            const int s = step_of(v);
            if (s >= kBins || v <= x_floor) return;          // (tokens at the floor are added below)
            if (!weigh) {
                atomicAdd(&sh.hist[0][s], 1u);
            } else {   // a 64-bit sum as two words: the carry goes with the high one
                const u64 w = row.whole(v);
                const unsigned l = static_cast<unsigned>(w), old = atomicAdd(&sh.hist[0][s], l);
                const unsigned h = static_cast<unsigned>(w >> 32) + (old + l < old ? 1u : 0u);
                if (h) atomicAdd(&sh.hist[1][s], h);
            }
        });
        cluster_sync();
        // this CTA's share of the steps, a step per thread, added up over the cluster
        u64 val = 0;
        const int my_step = static_cast<int>(rank) * kShare + tid;
        if (tid < kShare) {
            unsigned l[kC], h[kC];
#pragma unroll
            for (int r = 0; r < kC; r++) {
                l[r] = ld_u32(peer(&sh.hist[0][my_step], r));
                h[r] = weigh ? ld_u32(peer(&sh.hist[1][my_step], r)) : 0u;
            }
#pragma unroll
            for (int r = 0; r < kC; r++) val += l[r] + (static_cast<u64>(h[r]) << 32);
            if (fk && step_of(logit_of_key(fk)) == my_step) val += ft * fw;   // top-k's last key: its kept ties
        }
        u64 mine, before = cta_prefix(val, sh.red, mine);
        if (tid < kC) st_u64(peer(&sh.sum[0][rank], tid), mine);
        cluster_sync();
        u64 all = 0;
#pragma unroll
        for (int r = 0; r < kC; r++) {
            if (r < static_cast<int>(rank)) before += sh.sum[0][r];
            all += sh.sum[0][r];
        }
        // the step with the k-th token, or the one where top-p's sum is reached
        const u64 need = weigh ? max(part_of(p24, all), 1ull) : min(static_cast<u64>(k), all);
        if (before < need && need <= before + val)
            for (int r = 0; r < kC; r++) {
                st_u32(peer(&sh.step, r), my_step);
                st_u64(peer(&sh.before, r), before);
            }
        cluster_sync();
        const int step = static_cast<int>(sh.step);
        // the smallest logits down to the step, and down to the one before: 32 candidates at a time (step_of falls with
        // the logit), so that the passes below only compare
        auto least = [&](int st) {
            u64 l = 0, h = key_of(m);                        // step_of(h) <= st; of l - 1, if there is one, > st
            while (l < h) {
                const u64 d = h - l, mid = l + d * lane / 32;
                const float xv = logit_of_key(static_cast<uint32_t>(mid));
                const unsigned ok = __ballot_sync(0xffffffffu, xv == xv && step_of(xv) <= st);   // lanes from the first on
                const int f = ok ? __ffs(ok) - 1 : 32;
                const u64 nh = f < 32 ? l + d * f / 32 : h;
                l = f > 0 ? l + d * (f - 1) / 32 + 1 : l;
                h = nh;
            }
            return logit_of_key(static_cast<uint32_t>(h));
        };
        const float x_le = fmaxf(least(step), x_floor), x_lt = step > 0 ? least(step - 1) : INFINITY;
        const bool top_step = step == 0;                     // (x_lt then bounds nothing)
        auto in_le = [&](float v) { return v >= x_le && v > x_floor; };
        auto in_eq = [&](float v) { return in_le(v) && (top_step || v < x_lt); };
        // how many tokens lie down to the step, and in it
        unsigned le = 0, eq = 0;
        each([&](int, float v) {
            le += in_le(v);
            eq += in_eq(v);
        });
        le = static_cast<unsigned>(cta_sum(le, sh.red));
        eq = static_cast<unsigned>(cta_sum(eq, sh.red));
        if (tid < kC) {
            st_u32(peer(&sh.cnt[0][rank], tid), le);
            st_u32(peer(&sh.cnt[1][rank], tid), eq);
        }
        if (tid == 0) sh.n_mine = 0;
        cluster_sync();
        unsigned n_le = 0, n_eq = 0, o_le = 0, o_eq = 0;     // in all, and of the CTAs before this one
#pragma unroll
        for (int r = 0; r < kC; r++) {
            if (r == static_cast<int>(rank)) {
                o_le = n_le;
                o_eq = n_eq;
            }
            n_le += sh.cnt[0][r];
            n_eq += sh.cnt[1][r];
        }
        // (after a top-k the floor's ties are not among the candidates: no shortcut there)
        const bool small = n_le <= kCap && !(weigh && by_k);
        if (!small && n_eq > kCap) {
            bisect(need, weigh, fk, ft);
            continue;
        }
        each([&](int i, float v) {
            if (small ? in_le(v) : in_eq(v)) {
                const unsigned at = (small ? o_le : o_eq) + atomicAdd(&sh.n_mine, 1u);
                st_u64(peer(&sh.cand[at], 0), as_cand(i, v));
            }
        });
        cluster_sync();
        if (small) {                                         // the first CTA has all that is needed
            if (rank == 0) solve(static_cast<int>(n_le), [&](int i) { return sh.cand[i]; }, weigh, need);
            return;
        }
        if (rank == 0) {
            // the threshold inside the step; past its tokens lies the floor
            int n2 = 32;
            const int nc = static_cast<int>(n_eq);
            while (n2 < nc) n2 <<= 1;
            for (int i = nc + tid; i < n2; i += kNT) sh.cand[i] = ~0ull;
            cta_sort(sh.cand, n2);
            const int per = max(1, n2 / kNT), i0 = tid * per;
            auto measure_of = [&](u64 v) { return weigh ? row.whole(logit_of_key(~static_cast<uint32_t>(v >> 32))) : 1ull; };
            u64 w = 0, tot;
            for (int i = i0; i < min(i0 + per, nc); i++) w += measure_of(sh.cand[i]);
            u64 at = sh.before + cta_prefix(w, sh.red, tot);
            if (tid == 0) sh.thr = 0;
            __syncthreads();
            const u64 at0 = at;
            for (int i = i0; i < min(i0 + per, nc); i++) {
                const u64 x = measure_of(sh.cand[i]);
                if (at < need && need <= at + x) sh.thr = ~static_cast<uint32_t>(sh.cand[i] >> 32);
                at += x;
            }
            __syncthreads();
            uint32_t key_t = sh.thr;
            u64 n_t = 0;
            at = at0;
            for (int i = i0; i < min(i0 + per, nc); i++) {
                if (~static_cast<uint32_t>(sh.cand[i] >> 32) == key_t && at < need) n_t++;
                at += measure_of(sh.cand[i]);
            }
            n_t = cta_sum(n_t, sh.red);
            if (key_t == 0) {                                // reached by ties at the floor only
                key_t = fk;
                n_t = min((need - sh.before - tot + fw - 1) / max(fw, 1ull), ft);
            }
            __syncthreads();
            if (tid < kC) {
                st_u32(peer(&sh.thr, tid), key_t);
                st_u64(peer(&sh.ties, tid), n_t);
            }
        }
        cluster_sync();
        thr = sh.thr;
        ties = sh.ties;
    }
    // ---------------- the draw over all CTAs: per warp (its stretch of indexes) the kept weight above the threshold and
    // the tokens at it
    const u64 w_thr = thr ? row.whole(logit_of_key(thr)) : 0ull;
    const bool thr_ok = thr && row.weight(logit_of_key(thr)) >= mp;
    const float x_thr = thr ? logit_of_key(thr) : -INFINITY;
    auto part = [&](float v, u64 &s, unsigned &q) {
        const float w = row.weight(v);
        if (v > x_thr && w >= mp) s += whole_of(w);
        q += v == x_thr && thr_ok ? 1u : 0u;
    };
    {
        u64 s = 0;
        unsigned q = 0;
        each([&](int, float v) { part(v, s, q); });
        s = warp_sum64(s);
        q = __reduce_add_sync(0xffffffffu, q);
        if (lane == 0) {
            sh.ent[0][warp] = s;
            sh.ent[1][warp] = q;
        }
    }
    __syncthreads();
    if (warp < 2) {   // exclusive scans over the warps; the total after the last
        const u64 v = lane < kNW ? sh.ent[warp][lane] : 0ull, inc = warp_scan64(v);
        __syncwarp();
        if (lane <= kNW) sh.ent[warp][lane] = inc - v;   // (lane kNW: the total)
        const u64 all = __shfl_sync(0xffffffffu, inc, 31);
        if (lane < kC) {
            if (warp == 0) st_u64(peer(&sh.sum[0][rank], lane), all);
            else st_u32(peer(&sh.cnt[0][rank], lane), static_cast<unsigned>(all));
        }
    }
    cluster_sync();
    u64 s_all = 0, q_all = 0, s_me = 0, q_me = 0;
#pragma unroll
    for (int r = 0; r < kC; r++) {
        if (r == static_cast<int>(rank)) {
            s_me = s_all;
            q_me = q_all;
        }
        s_all += sh.sum[0][r];
        q_all += sh.cnt[0][r];
    }
    // the kept weight before a place with s above the threshold and q tokens at it before it
    auto kept = [&](u64 s, u64 q) { return s + min(q, ties) * w_thr; };
    const u64 total = kept(s_all, q_all), target = part_of(u24, total);
    u64 s0 = s_me + sh.ent[0][warp], q0 = q_me + sh.ent[1][warp];
    if (!(kept(s0, q0) <= target && target < kept(s_me + sh.ent[0][warp + 1], q_me + sh.ent[1][warp + 1]))) return;
    for (int i = first + 4 * lane; i < first + region; i += 128) {   // the warp that has the token: 128 at a time
        const float4 v = *reinterpret_cast<const float4 *>(xs + i);
        const float vs[4] = {v.x, v.y, v.z, v.w};
        u64 ls = 0;
        unsigned lq = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) part(vs[c], ls, lq);
        const u64 is = warp_scan64(ls), iq = warp_scan64(lq);
        u64 s = s0 + is - ls;
        unsigned q = static_cast<unsigned>(q0 + iq) - lq;
        s0 += __shfl_sync(0xffffffffu, is, 31);
        q0 += __shfl_sync(0xffffffffu, iq, 31);
        if (kept(s0, q0) <= target) continue;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const u64 b0 = kept(s, q);
            part(vs[c], s, q);
            if (b0 <= target && target < kept(s, q)) finish(lo + i + c, vs[c], total);
        }
        break;
    }
}

}  // namespace

cudaError_t launch_sample(const SampleArgs &a, cudaStream_t st) {
    // (a row up to 262144 logits fits eight CTAs' shared memory; beyond that it is read once per digit)
    if (a.n_vocab > kC * kSlice) return launch_pdl(k_sample, dim3(a.n_rows), dim3(kThreads), 0, st, a);
    const int region = ((a.n_vocab + kC * kNW - 1) / (kC * kNW) + 127) & ~127;
    const bool bulk = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.row_stride % 4 == 0;
    const cudaError_t e = allow_smem<k_sample_cluster>(kSlice * 4);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.n_rows) * kC);
    cfg.blockDim = dim3(kNT);
    cfg.dynamicSmemBytes = std::max(static_cast<size_t>(region) * kNW * 4, static_cast<size_t>(kCap) * 8);   // (solve sorts there)
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = kC;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    // (up to 163840 logits two CTAs fit an SM, and more than 32 clusters are more than one wave; beyond that one fits,
    // and 19 to 32 rows, more than a wave too, are taken in the order given)
    return cudaLaunchKernelEx(&cfg, k_sample_cluster, a, region, bulk, a.n_rows > 32 && a.n_rows <= kNT);
}

}  // namespace styx
