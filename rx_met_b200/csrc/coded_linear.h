// Product of 8-bit codes with an epilogue: the problem, and the kernels it is given to.
#pragma once

#include "common.h"

namespace rxmet {
namespace codedlinear {

struct Problem {
    int64_t rows;
    int inner, outer;
    const int8_t *codes;
    int64_t codesPitch;
    const float *scale;          // [rows]
    const int8_t *weight;
    int64_t weightPitch;
    const float *weightScale;    // [outer]
    const float *bias;           // [outer] or null
    int activation;
    const void *residual;        // [rows], type of out, or null
    int64_t residualPitch;
    int outType;
    void *out;                   // [rows][outer]
};

// Operands whose rows start on 16 bytes.
bool takesTensorCores(const Problem &p);
void launchTensorCores(const Problem &p, cudaStream_t st);

}  // namespace codedlinear
}  // namespace rxmet
