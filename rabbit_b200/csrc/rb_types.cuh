// rb_types.cuh -- activations of the cache-side operators in fp32, fp16 and
// bf16: vector loads and stores through fp32 registers, and the dispatch on a
// RABBIT_CUDA_F32 / F16 / BF16 argument.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/rabbit_cuda.h"

namespace rb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Eight elements; VEC: p is 16-byte aligned.
template <bool VEC, typename T>
__device__ __forceinline__ void load8(float (&d)[8], const T *p) {
    if constexpr (VEC) {
        uint4 w[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4 *>(p)[i];
        const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = to_f32(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = to_f32(p[i]);
    }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store8(T *p, const float (&d)[8]) {
    if constexpr (VEC) {
        uint4 w[sizeof(T) / 2];
        T *e = reinterpret_cast<T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(d[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(d[i]);
    }
}

// Bytes of an element, 0 for a code that is none.
inline int dtype_size(int dtype) {
    return dtype == RABBIT_CUDA_F32 ? 4 : dtype == RABBIT_CUDA_F16 || dtype == RABBIT_CUDA_BF16 ? 2 : 0;
}

// f(T()) for the element type of `dtype` (checked by the caller).
template <typename F>
inline auto with_dtype(int dtype, F &&f) {
    if (dtype == RABBIT_CUDA_F32) return f(float());
    if (dtype == RABBIT_CUDA_F16) return f(__half());
    return f(__nv_bfloat16());
}

}  // namespace rb
