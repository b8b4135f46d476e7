// Activations kept in 8 bits: a group's exponent, its codes, and the values that they stand for.
#pragma once

#include "element_types.cuh"
#include "rxmet_b200_gated.h"

namespace rxmet {
namespace kept {

constexpr int kGroup = RXMET_KEPT_GROUP;
constexpr int kBad = 127;   // exponent of a group that is not finite

inline int lowestExponent(int type) { return type == RXMET_TYPE_F16 ? -24 : -126; }
__host__ __device__ inline int groupsOf(int width) { return (width + kGroup - 1) / kGroup; }

// From the bits of a group's largest magnitude: the least e with which that is at most 127 * 2^e (127 = 1.984375 * 2^6).
__device__ __forceinline__ int exponentOf(uint32_t largest, int lowest) {
    if (largest >= 0x7f800000u) return kBad;
    return max(static_cast<int>(largest >> 23) - 133 + ((largest & 0x7fffffu) > 0x7e0000u ? 1 : 0), lowest);
}
// 2^e for e from -126 to 127.
__device__ __forceinline__ float powerOf(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float stepOf(int exponent) { return exponent == kBad ? __int_as_float(0x7fc00000) : powerOf(max(exponent, -126)); }

// Four codes of values times `inverse` = 2^-e: the sum with 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits.
__device__ __forceinline__ uint32_t codesOf(const float *v, float inverse) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(fmaf(v[i], inverse, 12582912.f));
    return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}
// What four codes stand for, by bytes of 2^23 + 128 + code.
__device__ __forceinline__ void valuesOf(uint32_t codes, float step, float *v) {
    const uint32_t raised = codes ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (__uint_as_float(__byte_perm(raised, 0x4b000000u, 0x7440 + i)) - 8388736.f) * step;
}

}  // namespace kept
}  // namespace rxmet
