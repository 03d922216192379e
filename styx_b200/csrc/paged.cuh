// paged.cuh -- addressing of a paged KV cache and its element types.
#pragma once

#include "../../include/styx_serve.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace styx {

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// rows of sequence b that the caches can hold: a length outside is clamped
// and reported
__device__ __forceinline__ int paged_len(const PagedKv &kv, int b, bool report) {
    const int n = __ldg(kv.lens + b);
    const long long most = static_cast<long long>(kv.max_pages) << kv.page_shift;
    if (n >= 0 && n <= most) return n;
    if (report) atomicExch(kv.err, kErrBadPos);
    return n < 0 ? 0 : static_cast<int>(most);
}

// element offset of (sequence b, kv head j, row r) in the pools; -1 for a
// page outside the pool.  r < max_pages * page_size.
__device__ __forceinline__ long long paged_off(const PagedKv &kv, int b, int j, int r) {
    const int page = __ldg(kv.table + static_cast<long long>(b) * kv.table_stride + (r >> kv.page_shift));
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(kv.n_pages)) return -1;
    const int in = (j << kv.page_shift) + (r & ((1 << kv.page_shift) - 1));
    return page * kv.page_stride + static_cast<long long>(in) * kv.hd;
}

}  // namespace styx
