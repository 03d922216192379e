// sample.cu -- temperature, top-k, top-p, min-p and the draw
// (styx_sample, include/styx_serve.h).
//
// The kept tokens are a prefix of the order (larger logit, lower index), so
// they are described by one threshold: all tokens whose key is above it and
// the first `ties` of those at it.  Weights are whole numbers (2^-40 of the
// largest one's), so every sum is exact whatever its order.
//
// k_sample_cluster (n_vocab <= 262144): a cluster of eight CTAs per row holds
// the row in shared memory, so the logits are read once.  One histogram over
// 2048 equal steps of log weight (tokens below e^-28 have weight 0 and take
// no part in anything) shows the step in which the threshold lies.  Where the
// tokens down to there are at most 512, they go to the cluster's first CTA,
// which sorts them and does the rest; else only that step's tokens go there,
// the threshold comes back, and every CTA sums its kept tokens for the draw.
// Only more than 512 tokens in one step (a flat row) are resolved by
// bisection of the key.  (The row in registers, 1024 threads of 64, spilled.)
//
// k_sample (larger vocabularies): one CTA per row, radix selection from L2.
#include <cuda_runtime.h>

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

struct Row {
    const float *x;
    float m, inv_t;
    bool hot;
    __device__ __forceinline__ float weight(float v) const {
        if (v == m) return 1.f;
        if (v == -INFINITY) return 0.f;   // an infinite temperature included
        return hot ? expf((v - m) * inv_t) : 0.f;
    }
    __device__ __forceinline__ u64 whole(float v) const { return static_cast<u64>(weight(v) * 0x1p40f); }
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
    row.inv_t = 1.0f / t;
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
constexpr int kBins = 4 * kNT, kCap = kNT;
constexpr float kBinScale = kBins / 28.f;
constexpr int kSlice = 32768;               // logits of a CTA at most
constexpr int kEnt = kSlice / (4 * kNT) * kNW;

struct Exchange {                           // what the cluster's CTAs write into each other
    float top[kC];
    u64 sum[2][kC];
    unsigned cnt[2][kC];
    unsigned n_cand, thr;
    u64 ties;
    u64 cand[kCap];                         // (inverted key << 32) | index: ascending = the order of the tokens
};
struct CtaShared {
    Exchange xc;
    unsigned cnt[kBins], lo[kBins], hi[kBins];
    u64 red[32], buf[kNT], ent[2][kEnt + 1];
    float redf[32];
    int step, upto;
    u64 before, in_step;
};

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
__device__ __forceinline__ uint4 ld_v4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ unsigned add_u32(uint32_t addr, unsigned v) {
    unsigned o;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(o) : "r"(addr), "r"(v) : "memory");
    return o;
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

// The CTA's values sorted ascending over its first n threads (a power of two,
// 32 or more; what lies beyond must be ~0): bitonic, strides below a warp by
// shuffles.
__device__ __forceinline__ u64 cta_sort(u64 v, int n, u64 *buf) {
    const int t = threadIdx.x;
    for (int size = 2; size <= n; size <<= 1) {
        const bool up = (t & size) == 0;
        for (int stride = size >> 1; stride >= 32; stride >>= 1) {
            buf[t] = v;
            __syncthreads();
            const u64 w = buf[t ^ stride];
            __syncthreads();
            v = ((t & stride) == 0) == up ? min(v, w) : max(v, w);
        }
        for (int stride = min(size >> 1, 16); stride; stride >>= 1) {
            const u64 w = __shfl_xor_sync(0xffffffffu, v, stride);
            v = ((t & stride) == 0) == up ? min(v, w) : max(v, w);
        }
    }
    return v;
}

__global__ void __launch_bounds__(kNT, 2) k_sample_cluster(SampleArgs a, int slice, bool vec) {
    extern __shared__ __align__(16) float xs[];   // [slice], cleaned
    __shared__ __align__(16) CtaShared sh;
    pdl_trigger();
    cl_arrive_relaxed();                          // the others have started: waited for before the first store to them
    Exchange &xc = sh.xc;
    const uint32_t rank = cluster_ctarank();
    const int b = blockIdx.x / kC, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = a.n_vocab;
    const int lo = static_cast<int>(rank) * slice, len = max(0, min(n - lo, slice));
    auto peer = [&](const void *p, uint32_t r) { return cl_map(smem_addr(p), r); };
    const uint4 z4 = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4 *>(sh.cnt)[tid] = z4;
    reinterpret_cast<uint4 *>(sh.lo)[tid] = z4;
    reinterpret_cast<uint4 *>(sh.hi)[tid] = z4;
    if (tid == 0) xc.n_cand = 0;
    pdl_wait();
    // ---------------- the slice, once; its maximum
    const float *src = a.logits + b * a.row_stride + lo;
    float m = -INFINITY;
#pragma unroll 5
    for (int i = 4 * tid; i < slice; i += 4 * kNT) {
        float4 v;
        if (vec && i + 4 <= len) {
            v = __ldcs(reinterpret_cast<const float4 *>(src + i));
        } else {
            v.x = i < len ? src[i] : -INFINITY;
            v.y = i + 1 < len ? src[i + 1] : -INFINITY;
            v.z = i + 2 < len ? src[i + 2] : -INFINITY;
            v.w = i + 3 < len ? src[i + 3] : -INFINITY;
        }
        v = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
        *reinterpret_cast<float4 *>(xs + i) = v;
        m = fmaxf(m, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
    Row row;
    row.x = nullptr;
    const float t = a.temperature ? a.temperature[b] : 1.f;
    row.hot = t > 0.f;
    row.inv_t = 1.0f / t;
    int k = a.top_k ? a.top_k[b] : 0;
    const float p = a.top_p ? fminf(a.top_p[b], 1.f) : 1.f;
    const u64 p24 = p > 0.f ? static_cast<u64>(rintf(p * 0x1p24f)) : 0ull;
    const float mp = a.min_p ? fminf(a.min_p[b], 1.f) : 0.f;   // the maximum always stays
    const u64 u24 = static_cast<u64>(fminf(fmaxf(a.u[b], 0.f), 0x1.fffffep-1f) * 0x1p24f);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sh.redf[warp] = m;
    __syncthreads();
    cl_wait();
    if (warp == 0) {
        m = lane < kNW ? sh.redf[lane] : -INFINITY;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane < kC) cl_st(peer(&xc.top[rank], lane), m);
    }
    cluster_sync();
    m = xc.top[0];
#pragma unroll
    for (int i = 1; i < kC; i++) m = fmaxf(m, xc.top[i]);
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
        for (int i = 4 * tid; i < slice; i += 4 * kNT) {
            const float4 v = *reinterpret_cast<const float4 *>(xs + i);
            f(i, v.x);
            f(i + 1, v.y);
            f(i + 2, v.z);
            f(i + 3, v.w);
        }
    };
    // the step of a token: kBins or more where the weight is 0
    const float bs = row.inv_t * kBinScale;
    auto step_of = [&](float v) {
        return v == m ? 0 : row.hot && v > -INFINITY ? static_cast<int>(fminf((m - v) * bs, kBins)) : kBins;
    };
    auto finish = [&](int i, float v, u64 total) {   // by the thread that has the token
        a.token[b] = i;
        if (a.logprob)
            a.logprob[b] = (v == m ? 0.f : (v - m) * row.inv_t) - logf(static_cast<float>(total) * 0x1p-40f);
    };
    uint32_t thr = 0;          // kept: keys above thr, and the first `ties` at it
    u64 ties = 0;
    if (by_k || by_p) {
        const bool weigh = !by_k;
        each([&](int, float v) {
            const int s = step_of(v);
            if (s >= kBins) return;
            atomicAdd(&sh.cnt[s], 1u);
            if (weigh) {   // a 64-bit sum as two words: the carry goes with the high one
                const u64 w = row.whole(v);
                const unsigned l = static_cast<unsigned>(w), old = atomicAdd(&sh.lo[s], l);
                const unsigned h = static_cast<unsigned>(w >> 32) + (old + l < old ? 1u : 0u);
                if (h) atomicAdd(&sh.hi[s], h);
            }
        });
        cluster_sync();
        // every CTA adds the eight histograms up, four steps per thread, and scans them from the top
        unsigned c4[4] = {0, 0, 0, 0};
        u64 w4[4] = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < kC; r++) {
            const uint4 v = ld_v4(peer(&sh.cnt[4 * tid], r));
            c4[0] += v.x, c4[1] += v.y, c4[2] += v.z, c4[3] += v.w;
        }
        if (weigh) {
#pragma unroll
            for (int r = 0; r < kC; r++) {
                const uint4 l = ld_v4(peer(&sh.lo[4 * tid], r)), h = ld_v4(peer(&sh.hi[4 * tid], r));
                w4[0] += l.x + (static_cast<u64>(h.x) << 32);
                w4[1] += l.y + (static_cast<u64>(h.y) << 32);
                w4[2] += l.z + (static_cast<u64>(h.z) << 32);
                w4[3] += l.w + (static_cast<u64>(h.w) << 32);
            }
        }
        u64 all_c, all_w = 0;
        u64 c0 = cta_prefix(static_cast<u64>(c4[0]) + c4[1] + c4[2] + c4[3], sh.red, all_c), w0 = 0;
        if (weigh) w0 = cta_prefix(w4[0] + w4[1] + w4[2] + w4[3], sh.red, all_w);
        // the step with the k-th token, or the one where top-p's sum is reached
        const u64 need = by_k ? min(static_cast<u64>(k), all_c) : max(part_of(p24, all_w), 1ull);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const u64 before = by_k ? c0 : w0, here = by_k ? c4[i] : w4[i];
            if (before < need && need <= before + here) {
                sh.step = 4 * tid + i;
                sh.upto = static_cast<int>(c0 + c4[i]);   // tokens down to here
                sh.before = before;
                sh.in_step = c4[i];
            }
            c0 += c4[i];
            w0 += w4[i];
        }
        __syncthreads();
        const int step = sh.step;
        const bool small = sh.upto <= kCap, gather = small || sh.in_step <= kCap;
        if (gather) {
            each([&](int i, float v) {
                const int s = step_of(v);
                if (small ? s <= step : s == step) {
                    const unsigned at = add_u32(peer(&xc.n_cand, 0), 1);
                    st_u64(peer(&xc.cand[at], 0),
                           (static_cast<u64>(~key_of(v)) << 32) | static_cast<unsigned>(lo + i));
                }
            });
            cluster_sync();
            if (small && rank != 0) return;          // the first CTA has all that is needed
            if (rank == 0) {
                const int nc = static_cast<int>(xc.n_cand);
                int n2 = 32;
                while (n2 < nc) n2 <<= 1;
                const bool in = tid < nc;
                const u64 v = cta_sort(in ? xc.cand[tid] : ~0ull, n2, sh.buf);
                const uint32_t key = ~static_cast<uint32_t>(v >> 32);
                const float xv = logit_of_key(key);
                const u64 w = in ? row.whole(xv) : 0ull;
                u64 tot;
                if (small) {
                    // sorted: top-k and top-p keep the first ones
                    const u64 before = cta_prefix(tid < k ? w : 0ull, sh.red, tot);
                    const u64 lim = !by_p ? ~0ull : by_k ? max(part_of(p24, tot), 1ull) : need;
                    const bool kept = in && tid < k && before < lim && row.weight(xv) >= mp;
                    const u64 total = cta_sum(kept ? w : 0ull, sh.red);
                    const u64 target = part_of(u24, total);
                    // the draw, in index order
                    const u64 z = cta_sort(kept ? ((v & 0xFFFFFFFFull) << 32) | key : ~0ull, n2, sh.buf);
                    const float zx = logit_of_key(static_cast<uint32_t>(z));
                    const u64 zw = z != ~0ull ? row.whole(zx) : 0ull;
                    const u64 zb = cta_prefix(zw, sh.red, tot);
                    if (zb <= target && target < zb + zw) finish(static_cast<int>(z >> 32), zx, total);
                    return;
                }
                // the threshold inside the step
                const u64 mine = by_k ? 1ull : w;
                const u64 before = sh.before + cta_prefix(in ? mine : 0ull, sh.red, tot);
                if (in && before < need && need <= before + mine) xc.thr = key;
                __syncthreads();
                const uint32_t key_t = xc.thr;
                const u64 eq = cta_sum(in && key == key_t && before < need ? 1ull : 0ull, sh.red);
                if (tid < kC) {
                    st_u32(peer(&xc.thr, tid), key_t);
                    st_u64(peer(&xc.ties, tid), eq);
                }
            }
            cluster_sync();
            thr = xc.thr;
            ties = xc.ties;
        }
        // Sum over the row's keys >= from of 1 or the weight; of the keys at floor_key only floor_ties count, none
        // below it.  Used by bisection: steps of more than kCap tokens, and top-p after a top-k of more than kCap.
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
                st_u64(peer(&xc.sum[slot][rank], tid), s);
                st_u32(peer(&xc.cnt[slot][rank], tid), static_cast<unsigned>(eq));
            }
            cluster_sync();
            u64 all = 0, q = 0;
#pragma unroll
            for (int r = 0; r < kC; r++) {
                all += xc.sum[slot][r];
                q += xc.cnt[slot][r];
            }
            return all + min(q, floor_ties) * (weights ? row.whole(logit_of_key(floor_key)) : 1ull);
        };
        // the largest key whose sum reaches lim, and how many of the tokens at it that takes
        auto bisect = [&](u64 lim, bool weights, uint32_t floor_key, u64 floor_ties) {
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
        if (!gather) bisect(need, weigh, 0, 0);
        if (by_k && by_p && !small) {
            const uint32_t fk = thr;
            const u64 ft = ties;
            cluster_sync();
            const u64 tot = measure(fk, fk, ft, true, 0);
            cluster_sync();
            bisect(max(part_of(p24, tot), 1ull), true, fk, ft);
        }
    }
    // ---------------- the draw over all CTAs: per (round of 4 kNT logits, warp) the kept weight above the threshold
    // and the tokens at it, in index order
    const u64 w_thr = thr ? row.whole(logit_of_key(thr)) : 0ull;
    const bool thr_ok = thr && row.weight(logit_of_key(thr)) >= mp;
    const int rounds = (slice + 4 * kNT - 1) / (4 * kNT), ents = rounds * kNW;
    auto part = [&](float v, u64 &s, u64 &q) {
        const uint32_t key = key_of(v);
        if (key > thr) {
            const float w = row.weight(v);
            if (w >= mp) s += static_cast<u64>(w * 0x1p40f);
        }
        q += key == thr && thr_ok ? 1 : 0;
    };
    for (int e = 0; e < rounds; e++) {
        const int i = 4 * (e * kNT + tid);
        u64 s = 0, q = 0;
        if (i < slice) {
            const float4 v = *reinterpret_cast<const float4 *>(xs + i);
            part(v.x, s, q);
            part(v.y, s, q);
            part(v.z, s, q);
            part(v.w, s, q);
        }
        s = warp_sum64(s);
        const unsigned qs = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(q));
        if (lane == 0) {
            sh.ent[0][e * kNW + warp] = s;
            sh.ent[1][e * kNW + warp] = qs;
        }
    }
    __syncthreads();
    if (warp < 2) {   // exclusive scans of the entries; the total after the last
        u64 run = 0;
        for (int i0 = 0; i0 < ents; i0 += 32) {
            const u64 v = i0 + lane < ents ? sh.ent[warp][i0 + lane] : 0ull;
            const u64 inc = warp_scan64(v);
            __syncwarp();
            if (i0 + lane < ents) sh.ent[warp][i0 + lane] = run + inc - v;
            run += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) sh.ent[warp][ents] = run;
        if (lane < kC) {
            if (warp == 0) st_u64(peer(&xc.sum[0][rank], lane), run);
            else st_u32(peer(&xc.cnt[0][rank], lane), static_cast<unsigned>(run));
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
        s_all += xc.sum[0][r];
        q_all += xc.cnt[0][r];
    }
    // the kept weight before a place with s above the threshold and q tokens at it before it
    auto kept = [&](u64 s, u64 q) { return s + min(q, ties) * w_thr; };
    const u64 total = kept(s_all, q_all), target = part_of(u24, total);
    for (int e = 0; e < rounds; e++) {
        const int at = e * kNW + warp;
        u64 s = s_me + sh.ent[0][at], q = q_me + sh.ent[1][at];
        if (!(kept(s, q) <= target && target < kept(s_me + sh.ent[0][at + 1], q_me + sh.ent[1][at + 1]))) continue;
        const int i = 4 * (e * kNT + tid);
        float4 v = i < slice ? *reinterpret_cast<const float4 *>(xs + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        u64 ls = 0, lq = 0;
        part(v.x, ls, lq);
        part(v.y, ls, lq);
        part(v.z, ls, lq);
        part(v.w, ls, lq);
        s += warp_scan64(ls) - ls;
        q += warp_scan64(lq) - lq;
        const float vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const u64 b0 = kept(s, q);
            part(vs[c], s, q);
            if (b0 <= target && target < kept(s, q)) finish(lo + i + c, vs[c], total);
        }
    }
}

}  // namespace

cudaError_t launch_sample(const SampleArgs &a, cudaStream_t st) {
    // (a row up to 262144 logits fits eight CTAs' shared memory; beyond that it is read once per digit)
    if (a.n_vocab > kC * kSlice) return launch_pdl(k_sample, dim3(a.n_rows), dim3(kThreads), 0, st, a);
    const int slice = (((a.n_vocab + kC - 1) / kC) + 3) & ~3;
    const bool vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.row_stride % 4 == 0;
    const cudaError_t e = cudaFuncSetAttribute(k_sample_cluster, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlice * 4);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.n_rows) * kC);
    cfg.blockDim = dim3(kNT);
    cfg.dynamicSmemBytes = static_cast<size_t>(slice) * 4;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = kC;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_sample_cluster, a, slice, vec);
}

}  // namespace styx
