// Linear attention with a decay for each head: one pass of the operator, in the roles that the forward and the gradients give it.
#pragma once

#include <cmath>

#include "common.h"
#include "rxmet_b200_mixer.h"

namespace rxmet {
namespace decayed {

constexpr int kMaxDim = 128;
constexpr int kMaxTokens = 1 << 30;   // places of tokens, rounded up to chunks and segments, are counted in 32 bits

// Forward in time:   S = decay S + k v',  o = outScale q S.
// Reverse in time:   S = S + k v',  o = outScale q S,  S = decay S   (from the last token to the first).
// The gradients are passes too.  With G the gradient of the state, G = decay G + scale q do' from the end on:
//   dq = scale S do:  forward, (do, v, k) for (q, k, v), the state transposed;
//   dv = k G:         reverse, (k, q, do);      dk = G v:  reverse, (v, do, q), transposed;
// where the scale is taken out of G, so that the state's gradient comes in divided by it and goes out multiplied.
struct Pass {
    int batch, tokens, heads, key, value;   // key: width of q and k, value: width of v and out
    rxmet_head_tensor q, k, v;              // without data, and strides of 0: zeros
    const float *logDecay;
    const int32_t *lengths;
    bool reverse;
    float outScale;
    // Element (b, h, i, j) of the state, i along key: at (b heads + h) key value + i rowStride + j colStride, times its scale.
    const float *stateIn;
    float *stateOut;
    int stateRow, stateCol;
    float inScale, finalScale;
    void *out;              // [batch][tokens][heads][value] of the type of q, or of 32 bits with outFloat
    bool outFloat;
};

void launchRecurrent(const Pass &p, int type, cudaStream_t st);

// One token forward, states of whole 16-byte groups.
bool takesStep(const Pass &p);
void launchStep(const Pass &p, int type, cudaStream_t st);

// Chunks of 128 tokens on tensor cores, for 16-bit tensors that TMA can copy.  Few heads are cut into segments along time, whose states need a workspace.
constexpr int kChunkTokens = 128;
struct ChunkPlan {
    bool taken;   // by size and type
    int segments, segmentChunks;
    size_t stateFloats(const Pass &p) const { return segments > 1 ? static_cast<size_t>(p.batch) * p.heads * segments * p.key * p.value : 0; }
};
ChunkPlan planChunks(const Pass &p, int type);
bool chunksCanCopy(const Pass &p);
void launchChunks(const Pass &p, int type, const ChunkPlan &plan, float *states, cudaStream_t st);

}  // namespace decayed
}  // namespace rxmet
