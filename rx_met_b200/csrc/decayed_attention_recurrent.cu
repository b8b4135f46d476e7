// Linear attention with a decay for each head, token by token, in 32-bit floats.
//
// A warp owns 32 columns of a head's state, a CTA all of them: lane = one of eight groups of four columns x one of four groups of rows, so that a row
// of the state is read and written 128 bytes at a time and the state stays in registers over all tokens.  Rows are dealt to the row groups four at a time,
// which keeps the four 16-byte reads of a key apart in shared memory.  Tokens come to shared memory sixteen at a time.
//
// Bound: the state's bytes for single tokens; the multiply-adds for many (4 operations an element of the state and token).
#include "decayed_attention.h"
#include "dependent_launch.cuh"
#include "element_types.cuh"

namespace rxmet {
namespace decayed {
namespace {

constexpr int kStage = 16;   // tokens in shared memory

template <class T>
struct Tokens {
    const T *data;
    int64_t strideT;
    __device__ __forceinline__ Tokens(const rxmet_head_tensor &t, int b, int h, int heads)
        : data(static_cast<const T *>(t.data) + b * t.stride_b + static_cast<int64_t>(h / (heads / t.heads)) * t.stride_h), strideT(t.stride_t) {}
};

// KEYS: rows of the state that the registers hold (64 or 128), those beyond `key` as zeros.
template <class T, int KEYS>
__global__ void __launch_bounds__(128) decayedRecurrent(const __grid_constant__ Pass p) {
    constexpr int kGroups = KEYS / 16;   // groups of four rows that a lane owns
    __shared__ __align__(16) float sq[kStage][KEYS], sk[kStage][KEYS], sv[kStage][kMaxDim];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int col = warp * 32 + (lane & 7) * 4, rowGroup = lane >> 3;
    waitForPredecessor();
    const int length = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
    // The decay as a sum of two floats: rounded to one, its error would grow with every token that a state remembers (2e-4 of the state over 4096 tokens
    // at a memory of 512).
    const double exact = exp(static_cast<double>(p.logDecay[h]));
    const float decay = static_cast<float>(exact), rest = static_cast<float>(exact - decay);
    const Tokens<T> q(p.q, b, h, p.heads), k(p.k, b, h, p.heads), v(p.v, b, h, p.heads);
    const size_t head = (static_cast<size_t>(b) * p.heads + h) * p.key * p.value;

    float s[kGroups][4][4];
    const bool groups = p.stateCol == 1 && p.value % 4 == 0 && (reinterpret_cast<uintptr_t>(p.stateIn) | reinterpret_cast<uintptr_t>(p.stateOut)) % 16 == 0;   // 16 bytes at a time
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * i + 4 * rowGroup + r;
            if (groups) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p.stateIn && row < p.key && col < p.value) v = *reinterpret_cast<const float4 *>(p.stateIn + head + static_cast<size_t>(row) * p.stateRow + col);
                s[i][r][0] = v.x * p.inScale;
                s[i][r][1] = v.y * p.inScale;
                s[i][r][2] = v.z * p.inScale;
                s[i][r][3] = v.w * p.inScale;
                continue;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
                s[i][r][c] = p.stateIn && row < p.key && col + c < p.value ? p.inScale * p.stateIn[head + static_cast<size_t>(row) * p.stateRow + static_cast<size_t>(col + c) * p.stateCol] : 0.f;
        }
    letDependentsStart();

    auto store = [&](int t, int c, float value) {
        if (!p.out || c >= p.value) return;
        const size_t at = ((static_cast<size_t>(b) * p.tokens + t) * p.heads + h) * p.value + c;
        if (p.outFloat) static_cast<float *>(p.out)[at] = value;
        else static_cast<T *>(p.out)[at] = fromFloat<T>(value);
    };
    for (int done = 0; done < length; done += kStage) {
        const int count = min(kStage, length - done);
        __syncthreads();
        // token i of the stage, in the order of the pass
        auto tokenOf = [&](int i) { return static_cast<int64_t>(p.reverse ? length - 1 - done - i : done + i); };
        for (int i = tid; i < count * KEYS; i += blockDim.x) {
            const int t = i / KEYS, d = i % KEYS;
            sq[t][d] = d < p.key ? toFloat(q.data[tokenOf(t) * q.strideT + d]) : 0.f;
            sk[t][d] = d < p.key ? toFloat(k.data[tokenOf(t) * k.strideT + d]) : 0.f;
        }
        for (int i = tid; i < count * kMaxDim; i += blockDim.x) {
            const int t = i / kMaxDim, d = i % kMaxDim;
            sv[t][d] = d < p.value ? toFloat(v.data[tokenOf(t) * v.strideT + d]) : 0.f;
        }
        __syncthreads();
        for (int t = 0; t < count; ++t) {
            const float4 vv = *reinterpret_cast<const float4 *>(&sv[t][col]);
            float o[4] = {};
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const float4 kk = *reinterpret_cast<const float4 *>(&sk[t][16 * i + 4 * rowGroup]), qq = *reinterpret_cast<const float4 *>(&sq[t][16 * i + 4 * rowGroup]);
                const float ks[4] = {kk.x, kk.y, kk.z, kk.w}, qs[4] = {qq.x, qq.y, qq.z, qq.w}, vs[4] = {vv.x, vv.y, vv.z, vv.w};
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float before = s[i][r][c], kv = ks[r] * vs[c];
                        const float now = p.reverse ? before + kv : fmaf(before, decay, fmaf(before, rest, kv));
                        o[c] = fmaf(qs[r], now, o[c]);
                        s[i][r][c] = p.reverse ? fmaf(now, decay, now * rest) : now;
                    }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                o[c] += __shfl_xor_sync(0xffffffffu, o[c], 8);
                o[c] += __shfl_xor_sync(0xffffffffu, o[c], 16);
            }
            // each row group stores one of the four columns
            const float mine = rowGroup == 0 ? o[0] : rowGroup == 1 ? o[1] : rowGroup == 2 ? o[2] : o[3];
            store(static_cast<int>(tokenOf(t)), col + rowGroup, mine * p.outScale);
        }
    }
    for (int t = length; t < p.tokens; ++t) store(t, col + rowGroup, 0.f);
    if (!p.stateOut) return;
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * i + 4 * rowGroup + r;
            if (groups) {
                if (row < p.key && col < p.value)
                    *reinterpret_cast<float4 *>(p.stateOut + head + static_cast<size_t>(row) * p.stateRow + col) =
                        make_float4(s[i][r][0] * p.finalScale, s[i][r][1] * p.finalScale, s[i][r][2] * p.finalScale, s[i][r][3] * p.finalScale);
                continue;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (row < p.key && col + c < p.value) p.stateOut[head + static_cast<size_t>(row) * p.stateRow + static_cast<size_t>(col + c) * p.stateCol] = s[i][r][c] * p.finalScale;
        }
}

}  // namespace

void launchRecurrent(const Pass &p, int type, cudaStream_t st) {
    const dim3 grid(p.heads, p.batch);
    const int threads = (p.value + 31) / 32 * 32;
    withType(type, [&](auto t) {
        using T = decltype(t);
        {
            KernelTimer timer__("decayedRecurrent", st);
            if (p.key <= 64) launchDependent(decayedRecurrent<T, 64>, grid, threads, 0, st, p);
            else launchDependent(decayedRecurrent<T, 128>, grid, threads, 0, st, p);
        }
        afterLaunch("decayedRecurrent");
    });
}

}  // namespace decayed
}  // namespace rxmet
