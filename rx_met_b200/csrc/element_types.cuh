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

// Two 32-bit floats in one operation each.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pairOf(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Pair pairOf(uint32_t a, uint32_t b) { return pairOf(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 floatsOf(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Two neighbours of a 16-bit type in one word.
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <class T>
__device__ __forceinline__ uint32_t pack2(Pair p) {
    const float2 v = floatsOf(p);
    return pack2<T>(v.x, v.y);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }

// A word of the current device that kernels set where a bounded wait gave up.  The results of that call are not to be used: some may be missing, some made from what was not there yet.
int *waitStatus();

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
