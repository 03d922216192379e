// paged_attn.cu -- attention of one new token per sequence over a paged KV
// cache (styx_paged_attend, include/styx_serve.h).
#include <cuda_runtime.h>

#include <cstdint>

#include "paged.cuh"

namespace styx {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kHeads = 8;        // q heads of a CTA
constexpr int kPerLane = 8;      // elements of a row per lane: head_dim <= 256

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// CTA (sequence, kv head, group of 8 q heads): a row per warp at a time, the
// running maximum, sum and output of every head in registers; the warps'
// states joined in shared memory at the end.
template <class T>
__global__ void __launch_bounds__(kThreads) k_paged_attend(PagedAttendArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float sq[kHeads][256];
    __shared__ float sm[kWarps][kHeads], sl[kWarps][kHeads];
    __shared__ float so[kWarps][256];
    const PagedKv &kv = a.kv;
    const int b = blockIdx.x, j = blockIdx.y, g0 = blockIdx.z * kHeads, ng = min(kHeads, a.gqa - g0);
    const int hd = kv.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = paged_len(kv, b, threadIdx.x == 0 && j == 0 && g0 == 0);
    const int first = a.window > 0 && a.window < n ? n - a.window : 0;
    const long long h0 = static_cast<long long>(b) * a.n_heads + j * a.gqa + g0;   // global index of the first head
    for (int i = threadIdx.x; i < ng * hd; i += kThreads) sq[i / hd][i % hd] = a.q[h0 * hd + i] * (a.scale * 1.4426950408889634f);
    __syncthreads();
    float m[kHeads], l[kHeads], o[kHeads][kPerLane];
#pragma unroll
    for (int g = 0; g < kHeads; g++) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int i = 0; i < kPerLane; i++) o[g][i] = 0.f;
    }
    float *scores = a.scores + (static_cast<long long>(b) * kv.n_kv + j) *
                                   (static_cast<long long>(kv.max_pages) << kv.page_shift) * a.gqa + g0;
    for (int r = first + warp; r < n; r += kWarps) {
        const long long off = paged_off(kv, b, j, r);
        if (off < 0 && lane == 0) atomicExch(kv.err, kErrBadPos);
        float kr[kPerLane], vr[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; i++) {
            const int c = lane + 32 * i;
            kr[i] = off >= 0 && c < hd ? to_f(static_cast<const T *>(kv.k)[off + c]) : 0.f;
            vr[i] = off >= 0 && c < hd ? to_f(static_cast<const T *>(kv.v)[off + c]) : 0.f;
        }
#pragma unroll
        for (int g = 0; g < kHeads; g++) {
            if (g < ng) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < kPerLane; i++)
                    if (lane + 32 * i < hd) s += kr[i] * sq[g][lane + 32 * i];
                s = off >= 0 ? warp_sum(s) : -INFINITY;
                if (a.acc_out && lane == 0) scores[static_cast<long long>(r) * a.gqa + g] = s;
                if (s > -INFINITY) {
                    const float mn = fmaxf(m[g], s), f = exp2f(m[g] - mn), p = exp2f(s - mn);
                    m[g] = mn;
                    l[g] = l[g] * f + p;
#pragma unroll
                    for (int i = 0; i < kPerLane; i++) o[g][i] = o[g][i] * f + p * vr[i];
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < kHeads; g++)
        if (lane == 0) {
            sm[warp][g] = m[g];
            sl[warp][g] = l[g];
        }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kHeads; g++) {
        if (g >= ng) break;
        float M = -INFINITY, L = 0.f;
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, sm[w][g]);
        for (int w = 0; w < kWarps; w++) L += sl[w][g] > 0.f ? exp2f(sm[w][g] - M) * sl[w][g] : 0.f;
        const float f = l[g] > 0.f ? exp2f(m[g] - M) / L : 0.f;
#pragma unroll
        for (int i = 0; i < kPerLane; i++)
            if (lane + 32 * i < hd) so[warp][lane + 32 * i] = f > 0.f ? o[g][i] * f : 0.f;
        __syncthreads();
        for (int c = threadIdx.x; c < hd; c += kThreads) {
            float s = 0.f;
            for (int w = 0; w < kWarps; w++) s += so[w][c];
            a.out[(h0 + g) * hd + c] = s;
        }
        if (threadIdx.x == 0) {
            if (a.lse) a.lse[h0 + g] = L > 0.f ? M * 0.6931471805599453f + logf(L) : -INFINITY;
            if (a.acc_out) {
                a.ml[2 * (h0 + g)] = M;
                a.ml[2 * (h0 + g) + 1] = L;
            }
        }
        __syncthreads();
    }
}

// acc_out[r] = (newest row: 0, else acc[r]) + the row's weights over the kv
// head's q heads, from the scores and every head's maximum and sum
__global__ void __launch_bounds__(256) k_paged_acc(PagedAttendArgs a) {
    pdl_trigger();
    pdl_wait();
    const PagedKv &kv = a.kv;
    const int b = blockIdx.y / kv.n_kv, j = blockIdx.y - b * kv.n_kv;
    const int n = paged_len(kv, b, false);
    const int first = a.window > 0 && a.window < n ? n - a.window : 0;
    const long long max_rows = static_cast<long long>(kv.max_pages) << kv.page_shift;
    const long long h0 = static_cast<long long>(b) * a.n_heads + j * a.gqa;
    const long long line = (static_cast<long long>(b) * kv.n_kv + j) * a.acc_stride;
    const float *scores = a.scores + (static_cast<long long>(b) * kv.n_kv + j) * max_rows * a.gqa;
    for (int r = blockIdx.x * 256 + threadIdx.x; r < n; r += gridDim.x * 256) {
        float w = 0.f;
        if (r >= first)
            for (int g = 0; g < a.gqa; g++) {
                const float L = a.ml[2 * (h0 + g) + 1];
                if (L > 0.f) w += exp2f(scores[static_cast<long long>(r) * a.gqa + g] - a.ml[2 * (h0 + g)]) / L;
            }
        a.acc_out[line + r] = r == n - 1 ? w : a.acc[line + r] + w;
    }
}

}  // namespace

cudaError_t launch_paged_attend(const PagedAttendArgs &a, cudaStream_t st) {
    const dim3 grid(a.kv.n_seqs, a.kv.n_kv, (a.gqa + kHeads - 1) / kHeads), block(kThreads);
    cudaError_t e;
    if (a.kv.dtype == STYX_F16) e = launch_pdl(k_paged_attend<__half>, grid, block, 0, st, a);
    else if (a.kv.dtype == STYX_BF16) e = launch_pdl(k_paged_attend<__nv_bfloat16>, grid, block, 0, st, a);
    else e = launch_pdl(k_paged_attend<float>, grid, block, 0, st, a);
    return e;
}

cudaError_t launch_paged_acc(const PagedAttendArgs &a, cudaStream_t st) {
    const long long max_rows = static_cast<long long>(a.kv.max_pages) << a.kv.page_shift;
    const dim3 ga(static_cast<unsigned>(max_rows < 64 * 256 ? (max_rows + 255) / 256 : 64),
                  static_cast<unsigned>(a.kv.n_seqs) * a.kv.n_kv);
    return launch_pdl(k_paged_acc, ga, dim3(256), 0, st, a);
}

}  // namespace styx
