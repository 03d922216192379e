// paged.cuh -- addressing of a paged KV cache and its element types.
#pragma once

#include "../../include/styx_serve.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace styx {

// Loads of what an earlier kernel may have written.  (__ldg and __ldcg carry no
// order with respect to griddepcontrol.wait: the compiler may move them above
// it, to where the earlier kernel's stores are not yet visible.)
template <class T>
__device__ __forceinline__ T ld_now(const T *p) {
    return *p;
}
__device__ __forceinline__ uint32_t ld_cg(const uint32_t *p) {   // from L2
    uint32_t v;
    asm volatile("ld.global.cg.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ int32_t ld_cg(const int32_t *p) {
    return static_cast<int32_t>(ld_cg(reinterpret_cast<const uint32_t *>(p)));
}
__device__ __forceinline__ float ld_cg(const float *p) { return __uint_as_float(ld_cg(reinterpret_cast<const uint32_t *>(p))); }
__device__ __forceinline__ float4 ld_cg(const float4 *p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "l"(p)
                 : "memory");
    return v;
}

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
    const int n = ld_now(kv.lens + b);
    const long long most = static_cast<long long>(kv.max_pages) << kv.page_shift;
    if (n >= 0 && n <= most) return n;
    if (report) atomicExch(kv.err, kErrBadPos);
    return n < 0 ? 0 : static_cast<int>(most);
}

// element offset of (sequence b, kv head j, row r) in the pools; -1 for a
// page outside the pool.  r < max_pages * page_size.
__device__ __forceinline__ long long paged_off(const PagedKv &kv, int b, int j, int r) {
    const int page = ld_now(kv.table + static_cast<long long>(b) * kv.table_stride + (r >> kv.page_shift));
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(kv.n_pages)) return -1;
    const int in = (j << kv.page_shift) + (r & ((1 << kv.page_shift) - 1));
    return page * kv.page_stride + static_cast<long long>(in) * kv.hd;
}

}  // namespace styx
