// Activations in 32-bit floats, bfloat16 and half: conversions and 16-byte accesses shared by the token mixer's kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "common.h"
#include "rxmet_b200_mixer.h"

namespace rxmet {

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float toFloat(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T fromFloat(float v);
template <>
__device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }

// W elements that are loaded and stored at once (16 bytes, or one element where alignment allows no more).
template <class T, int W>
struct alignas(W * sizeof(T)) Pack {
    T v[W];
};

inline size_t typeBytes(int type) { return type == RXMET_TYPE_F32 ? 4 : 2; }

// f(T{}) for the element type.
template <class F>
void withType(int type, F f) {
    if (type == RXMET_TYPE_F32) f(float{});
    else if (type == RXMET_TYPE_BF16) f(__nv_bfloat16{});
    else if (type == RXMET_TYPE_F16) f(__half{});
    else fail(RXMET_ERR_INVALID_ARGUMENT, "unknown element type %d", type);
}

}  // namespace rxmet
