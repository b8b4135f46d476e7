// Epilogue of the products of 8-bit codes.
#pragma once

#include "coded_linear.h"
#include "element_types.cuh"

namespace rxmet {
namespace codedlinear {

__device__ __forceinline__ float activate(float v, int activation) {
    if (activation == RXMET_ACTIVATION_RELU) return v < 0.f ? 0.f : v;   // keeps a NaN
    if (activation == RXMET_ACTIVATION_SILU) return v / (1.f + expf(-v));
    if (activation == RXMET_ACTIVATION_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    return v;
}

// What an output channel needs: its scale and bias.
struct Channel {
    float scale, bias;
    __device__ __forceinline__ Channel(const Problem &p, int n) : scale(p.weightScale[n]), bias(p.bias ? p.bias[n] : 0.f) {}
    // The exact integer sum is rounded to 32-bit float once; every further operation rounds once.
    __device__ __forceinline__ float value(int32_t sum, float rowScale, int activation) const {
        return activate(fmaf(static_cast<float>(sum) * rowScale, scale, bias), activation);
    }
};

}  // namespace codedlinear
}  // namespace rxmet
