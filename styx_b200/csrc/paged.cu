// paged.cu -- rows into and out of a paged KV cache (include/styx_serve.h):
//
//   k_paged_append   per-head RMSNorm, RoPE and the rounded K / V rows
//   k_evict_select   the rows that stay, and the row each place is filled from
//   k_evict_move     K, V, weight and position of the rows that move
#include <cuda_runtime.h>

#include <cstdint>

#include "paged.cuh"

namespace styx {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// CTA (token t, head h): h < n_heads a q head, else kv head h - n_heads.
// Thread i < hd/2 owns the pair (i, i + hd/2).
template <class T>
__global__ void __launch_bounds__(128) k_paged_append(PagedAppendArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float red[4];
    const PagedKv &kv = a.kv;
    const int rows = a.n_heads + kv.n_kv, hd = kv.hd, half = hd >> 1, i = threadIdx.x;
    const int t = blockIdx.x / rows, h = blockIdx.x - t * rows;
    const bool is_q = h < a.n_heads;
    const int head = is_q ? h : h - a.n_heads;
    const int b = a.seq ? a.seq[t] : t;
    if (static_cast<unsigned>(b) >= static_cast<unsigned>(kv.n_seqs)) {
        if (i == 0) atomicExch(kv.err, kErrBadPos);
        if (is_q)
            for (int c = i; c < hd; c += 128) a.q_out[(static_cast<long long>(t) * a.n_heads + head) * hd + c] = 0.f;
        return;
    }
    const int r = a.row ? a.row[t] : kv.lens[b] - 1;
    if (r < 0) {   // padding, or an empty slot
        if (is_q)
            for (int c = i; c < hd; c += 128) a.q_out[(static_cast<long long>(t) * a.n_heads + head) * hd + c] = 0.f;
        return;
    }
    const float *src = is_q ? a.q + t * a.q_stride + static_cast<long long>(head) * hd
                            : a.k + t * a.k_stride + static_cast<long long>(head) * hd;
    const float *w = is_q ? a.q_norm : a.k_norm;
    const bool on = i < half;
    float x0 = on ? src[i] : 0.f, x1 = on ? src[i + half] : 0.f;
    if (w) {
        float ss = warp_sum(x0 * x0 + x1 * x1);
        if ((i & 31) == 0) red[i >> 5] = ss;
        __syncthreads();
        ss = red[0] + red[1] + red[2] + red[3];
        const float scale = 1.0f / sqrtf(ss / static_cast<float>(hd) + a.eps);
        if (on) {
            x0 = x0 * scale * w[i];
            x1 = x1 * scale * w[i + half];
        }
    }
    long long off = 0;
    if (!is_q) {
        off = r < (static_cast<long long>(kv.max_pages) << kv.page_shift) ? paged_off(kv, b, head, r) : -1;
        if (off < 0) {
            if (i == 0) atomicExch(kv.err, kErrBadPos);
            return;
        }
        const float *vh = a.v + t * a.v_stride + static_cast<long long>(head) * hd;
        T *vrow = static_cast<T *>(kv.v) + off;
        for (int c = i; c < hd; c += 128) vrow[c] = from_f<T>(vh[c]);
    }
    if (on) {
        double sn, cs;
        sincos(static_cast<double>(a.pos[t]) * pow(a.theta_scale, static_cast<double>(i)), &sn, &cs);
        const float c = static_cast<float>(cs), s = static_cast<float>(sn);
        const float y0 = x0 * c - x1 * s, y1 = x0 * s + x1 * c;
        if (is_q) {
            float *o = a.q_out + (static_cast<long long>(t) * a.n_heads + head) * hd;
            o[i] = y0;
            o[i + half] = y1;
        } else {
            T *krow = static_cast<T *>(kv.k) + off;
            krow[i] = from_f<T>(y0);
            krow[i + half] = from_f<T>(y1);
        }
    }
}

// ------------------------------------------------------------ eviction
constexpr int kEvThreads = 1024;

// order of the weights as unsigned integers, larger first: protected rows
// above all, NaN as -inf, -0 as +0
__device__ __forceinline__ uint32_t evict_key(float acc, int pos, int next_pos, int n_recent, int n_sink) {
    if (static_cast<long long>(pos) >= static_cast<long long>(next_pos) - n_recent || pos < n_sink) return 0xFFFFFFFFu;
    if (acc != acc) acc = -INFINITY;
    const uint32_t b = __float_as_uint(acc + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);   // +inf: 0xFF800000, below the protected rows' key
}

__device__ __forceinline__ int block_scan(int v, int *warps, int &total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    if (lane == 31) warps[w] = s;
    __syncthreads();
    if (w == 0) {
        int x = warps[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += u;
        }
        warps[lane] = x;
    }
    __syncthreads();
    const int before = w ? warps[w - 1] : 0;
    total = warps[31];
    __syncthreads();
    return before + s - v;   // exclusive
}

// CTA (sequence, kv head): the key of the budget-th row by radix selection
// (four digits of 8 bits, from the top), then, tile by tile in row order,
// who stays: keys above the threshold, and the first rows at it.  Places
// (rows below the budget that leave) and movers (rows beyond that stay) are
// numbered as they come; place and mover i meet through the source list.
__global__ void __launch_bounds__(kEvThreads) k_evict_select(PagedEvictArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ unsigned hist[256];
    __shared__ int warps[32];
    __shared__ unsigned s_prefix;
    __shared__ int s_need;
    const PagedKv &kv = a.kv;
    const int b = blockIdx.x / kv.n_kv, j = blockIdx.x - b * kv.n_kv, tid = threadIdx.x;
    const int n = paged_len(kv, b, tid == 0 && j == 0);
    const int left = min(n, a.budget);
    const long long line = (static_cast<long long>(b) * kv.n_kv + j) * a.stride;
    const float *acc = a.acc + line;
    const int32_t *pos = a.pos + line;
    int32_t *src = a.src + (static_cast<long long>(b) * kv.n_kv + j) * a.budget;
    if (j == 0 && tid == 0) a.lens_out[b] = left;
    if (n <= a.budget) {
        for (int r = tid; r < n; r += kEvThreads) src[r] = r;
        return;
    }
    const int np = a.next_pos[b];
    if (tid == 0) {
        s_prefix = 0;
        s_need = left;
    }
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const unsigned prefix = s_prefix;
        const int need = s_need;
        for (int r = tid; r < n; r += kEvThreads) {
            const uint32_t k = evict_key(acc[r], pos[r], np, a.n_recent, a.n_sink);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            int above = 0, d = 255;
            for (; d > 0; d--) {
                if (above + static_cast<int>(hist[d]) >= need) break;
                above += static_cast<int>(hist[d]);
            }
            s_prefix = prefix | (static_cast<unsigned>(d) << shift);
            s_need = need - above;   // rows to take at the threshold digit
        }
        __syncthreads();
    }
    const unsigned thr = s_prefix;
    const int ties = s_need;   // of the rows equal to thr, the first `ties` stay
    int tie0 = 0, place0 = 0, mover0 = 0;
    // pass 1: places, in order, into the source list's tail end (as row
    // numbers); pass 2: movers.  Both lists are as long: the i-th mover goes
    // to the i-th place.
    for (int base = 0; base < n; base += kEvThreads) {
        const int r = base + tid;
        const bool in = r < n;
        const uint32_t k = in ? evict_key(acc[r], pos[r], np, a.n_recent, a.n_sink) : 0u;
        int tot;
        const int tr = block_scan(in && k == thr, warps, tot);
        const bool stay = in && (k > thr || (k == thr && tie0 + tr < ties));
        tie0 += tot;
        const bool place = in && r < left && !stay, mover = in && r >= left && stay;
        const int pr = block_scan(place, warps, tot);
        if (place) a.places[(static_cast<long long>(b) * kv.n_kv + j) * a.budget + place0 + pr] = r;
        place0 += tot;
        const int mr = block_scan(mover, warps, tot);
        if (in && r < left && stay) src[r] = r;
        __syncthreads();   // every place of a tile is listed before a later tile's mover reads it
        if (mover) src[a.places[(static_cast<long long>(b) * kv.n_kv + j) * a.budget + mover0 + mr]] = r;
        mover0 += tot;
    }
}

// CTA (sequence, kv head, part of the budget): weights and positions of the
// rows that stay, and K and V of those that move.  Sources lie at or beyond
// the budget, places below it, so no row is both.
template <class T>
__global__ void __launch_bounds__(256) k_evict_move(PagedEvictArgs a) {
    pdl_trigger();
    pdl_wait();
    const PagedKv &kv = a.kv;
    const int b = blockIdx.x / kv.n_kv, j = blockIdx.x - b * kv.n_kv;
    const int n = paged_len(kv, b, false);
    const int left = min(n, a.budget);
    const long long head = static_cast<long long>(b) * kv.n_kv + j;
    const int32_t *src = a.src + head * a.budget;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = blockIdx.y * 8 + warp; r < left; r += gridDim.y * 8) {
        const int s = src[r];
        if (lane == 0) {
            a.acc_out[head * a.stride + r] = a.acc[head * a.stride + s];
            a.pos_out[head * a.stride + r] = a.pos[head * a.stride + s];
        }
        if (s == r) continue;
        const long long from = paged_off(kv, b, j, s), to = paged_off(kv, b, j, r);
        if (from < 0 || to < 0) {
            if (lane == 0) atomicExch(kv.err, kErrBadPos);
            continue;
        }
        const T *k = static_cast<const T *>(kv.k), *v = static_cast<const T *>(kv.v);
        for (int c = lane; c < kv.hd; c += 32) {
            static_cast<T *>(kv.k)[to + c] = k[from + c];
            static_cast<T *>(kv.v)[to + c] = v[from + c];
        }
    }
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs &a, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.n_tokens) * (a.n_heads + a.kv.n_kv)), block(128);
    if (a.kv.dtype == STYX_F16) return launch_pdl(k_paged_append<__half>, grid, block, 0, st, a);
    if (a.kv.dtype == STYX_BF16) return launch_pdl(k_paged_append<__nv_bfloat16>, grid, block, 0, st, a);
    return launch_pdl(k_paged_append<float>, grid, block, 0, st, a);
}

cudaError_t launch_paged_evict(const PagedEvictArgs &a, cudaStream_t st) {
    const unsigned lines = static_cast<unsigned>(a.kv.n_seqs) * a.kv.n_kv;
    cudaError_t e = launch_pdl(k_evict_select, dim3(lines), dim3(kEvThreads), 0, st, a);
    if (e != cudaSuccess) return e;
    const dim3 grid(lines, static_cast<unsigned>(min(64, (a.budget + 7) / 8)));
    if (a.kv.dtype == STYX_F32) return launch_pdl(k_evict_move<uint32_t>, grid, dim3(256), 0, st, a);
    return launch_pdl(k_evict_move<uint16_t>, grid, dim3(256), 0, st, a);
}

}  // namespace styx
