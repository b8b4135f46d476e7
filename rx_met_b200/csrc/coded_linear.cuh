// Epilogue of the products of 8-bit codes.
#pragma once

#include "coded_linear.h"
#include "element_types.cuh"

namespace rxmet {
namespace codedlinear {

// One test of the activation for all values: a test for each would keep their chains of operations from running beside one another (160 cycles a value
// and warp instead of 20).
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int activation) {
    if (activation == RXMET_ACTIVATION_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];   // keeps a NaN
    } else if (activation == RXMET_ACTIVATION_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = __fdividef(v[j], 1.f + expf(-v[j]));
    } else if (activation == RXMET_ACTIVATION_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 0.5f * v[j] * (1.f + erff(v[j] * 0.70710678118654752f));
    }
}

// What an output channel needs: its scale and bias.
struct Channel {
    float scale, bias;
    __device__ __forceinline__ Channel(const Problem &p, int n) : scale(p.weightScale[n]), bias(p.bias ? p.bias[n] : 0.f) {}
    // In front of the activation.  The exact integer sum is rounded to a 32-bit float once; every further operation rounds once.
    __device__ __forceinline__ float value(int32_t sum, float rowScale) const { return fmaf(static_cast<float>(sum) * rowScale, scale, bias); }
};

}  // namespace codedlinear
}  // namespace rxmet
