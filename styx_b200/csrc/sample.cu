// sample.cu -- temperature, top-k, top-p, min-p and the draw
// (styx_sample, include/styx_serve.h).
//
// The kept tokens are a prefix of the order (larger logit, lower index), so
// they are described by one threshold: all tokens whose key is above it and
// the first `ties` of those at it.  Weights are whole numbers (2^-40 of the
// largest one's), so every sum is exact whatever its order.
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
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

}  // namespace

cudaError_t launch_sample(const SampleArgs &a, cudaStream_t st) {
    return launch_pdl(k_sample, dim3(a.n_rows), dim3(kThreads), 0, st, a);
}

}  // namespace styx
