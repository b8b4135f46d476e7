// Linear attention with a decay for each head, token by token, in 32-bit floats.
//
// A warp owns sixteen columns of a head's state, a CTA all of them: lane = one of four groups of four columns x one of eight groups of rows, and the state stays in
// registers over all tokens, two elements an operation.  Rows are dealt to the row groups four at a time, which keeps the eight 16-byte reads of a key apart in shared memory.
// Tokens come to shared memory sixteen at a time.  With 32 columns a warp, single operations and loads one after another a token of 64 heads of 128 took 2.2 us, now 0.6.
//
// Bound: the state's bytes for few tokens; issue for many (two packed operations an element of the state and token).
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
template <class T, int KEYS, bool Reverse>
__global__ void __launch_bounds__(256) decayedRecurrent(const __grid_constant__ Pass p) {
    constexpr int kGroups = KEYS / 32;   // groups of four rows that a lane owns
    __shared__ __align__(16) float sq[kStage][KEYS], sk[kStage][KEYS], sv[kStage][kMaxDim];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int col = warp * 16 + (lane & 3) * 4, rowGroup = lane >> 2;
    waitForPredecessor();
    const int length = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
    // The decay as a sum of two floats: rounded to one, its error would grow with every token that a state remembers (2e-4 of the state over 4096 tokens
    // at a memory of 512).
    const double exact = exp(static_cast<double>(p.logDecay[h]));
    const Pair decay = pairOf(static_cast<float>(exact), static_cast<float>(exact));
    const float left = static_cast<float>(exact - static_cast<float>(exact));
    const Pair rest = pairOf(left, left);
    const Tokens<T> q(p.q, b, h, p.heads), k(p.k, b, h, p.heads), v(p.v, b, h, p.heads);
    const size_t head = (static_cast<size_t>(b) * p.heads + h) * p.key * p.value;
    const bool groups = p.stateCol == 1 && p.value % 4 == 0 && (reinterpret_cast<uintptr_t>(p.stateIn) | reinterpret_cast<uintptr_t>(p.stateOut)) % 16 == 0;   // 16 bytes at a time

    Pair s[kGroups][4][2];
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 32 * i + 4 * rowGroup + r;
            const float *from = p.stateIn + head + static_cast<size_t>(row) * p.stateRow + static_cast<size_t>(col) * p.stateCol;
            float4 in = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.stateIn && row < p.key) {
                if (groups) {
                    if (col < p.value) in = *reinterpret_cast<const float4 *>(from);
                } else {
                    if (col < p.value) in.x = from[0];
                    if (col + 1 < p.value) in.y = from[p.stateCol];
                    if (col + 2 < p.value) in.z = from[2 * p.stateCol];
                    if (col + 3 < p.value) in.w = from[3 * p.stateCol];
                }
            }
            s[i][r][0] = pairOf(in.x * p.inScale, in.y * p.inScale);
            s[i][r][1] = pairOf(in.z * p.inScale, in.w * p.inScale);
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
        auto tokenOf = [&](int i) { return static_cast<int64_t>(Reverse ? length - 1 - done - i : done + i); };
        // eight loads in flight a thread: one after another, they took more time than the tokens
        auto fill = [&](const Tokens<T> &from, float *to, int dims, int width) {   // rows of `width` floats, zeros from `dims` on
            for (int i0 = tid; i0 < count * width; i0 += 8 * blockDim.x) {
                T in[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = i0 + e * blockDim.x, t = i / width, d = i - t * width;
                    in[e] = i < count * width && d < dims && from.data ? from.data[tokenOf(t) * from.strideT + d] : fromFloat<T>(0.f);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (i0 + e * static_cast<int>(blockDim.x) < count * width) to[i0 + e * blockDim.x] = toFloat(in[e]);
            }
        };
        fill(q, sq[0], p.key, KEYS);
        fill(k, sk[0], p.key, KEYS);
        fill(v, sv[0], p.value, kMaxDim);
        __syncthreads();
#pragma unroll 1
        for (int t = 0; t < count; ++t) {
            const float4 vv = *reinterpret_cast<const float4 *>(&sv[t][col]);
            const Pair vs[2] = {pairOf(vv.x, vv.y), pairOf(vv.z, vv.w)};
            Pair o[2] = {pairOf(0.f, 0.f), pairOf(0.f, 0.f)};
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const float4 kk = *reinterpret_cast<const float4 *>(&sk[t][32 * i + 4 * rowGroup]), qq = *reinterpret_cast<const float4 *>(&sq[t][32 * i + 4 * rowGroup]);
                const float ks[4] = {kk.x, kk.y, kk.z, kk.w}, qs[4] = {qq.x, qq.y, qq.z, qq.w};
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const Pair kr = pairOf(ks[r], ks[r]), qr = pairOf(qs[r], qs[r]);
                        Pair &state = s[i][r][c];
                        if constexpr (Reverse) {
                            const Pair now = fma2(kr, vs[c], state);
                            o[c] = fma2(qr, now, o[c]);
                            state = fma2(now, decay, mul2(now, rest));
                        } else {
                            state = fma2(state, decay, fma2(state, rest, mul2(kr, vs[c])));
                            o[c] = fma2(qr, state, o[c]);
                        }
                    }
            }
            float sums[4] = {floatsOf(o[0]).x, floatsOf(o[0]).y, floatsOf(o[1]).x, floatsOf(o[1]).y};
#pragma unroll
            for (int d = 4; d < 32; d *= 2)
#pragma unroll
                for (int c = 0; c < 4; ++c) sums[c] += __shfl_xor_sync(0xffffffffu, sums[c], d);
            // four of the row groups store one of the four columns each
            const float mine = rowGroup == 0 ? sums[0] : rowGroup == 1 ? sums[1] : rowGroup == 2 ? sums[2] : sums[3];
            if (rowGroup < 4) store(static_cast<int>(tokenOf(t)), col + rowGroup, mine * p.outScale);
        }
    }
    if (rowGroup < 4)
        for (int t = length; t < p.tokens; ++t) store(t, col + rowGroup, 0.f);
    if (!p.stateOut) return;
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 32 * i + 4 * rowGroup + r;
            if (row >= p.key) continue;
            float *to = p.stateOut + head + static_cast<size_t>(row) * p.stateRow + static_cast<size_t>(col) * p.stateCol;
            const float2 a = floatsOf(s[i][r][0]), c = floatsOf(s[i][r][1]);
            const float values[4] = {a.x * p.finalScale, a.y * p.finalScale, c.x * p.finalScale, c.y * p.finalScale};
            if (groups) {
                if (col < p.value) *reinterpret_cast<float4 *>(to) = make_float4(values[0], values[1], values[2], values[3]);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < p.value) to[static_cast<size_t>(e) * p.stateCol] = values[e];
        }
}

}  // namespace

void launchRecurrent(const Pass &p, int type, cudaStream_t st) {
    const dim3 grid(p.heads, p.batch);
    const int threads = (p.value + 15) / 16 * 32;
    withType(type, [&](auto t) {
        using T = decltype(t);
        auto run = [&](auto reverse) {
            constexpr bool Reverse = decltype(reverse)::value;
            KernelTimer timer__("decayedRecurrent", st);
            if (p.key <= 64) launchDependent(decayedRecurrent<T, 64, Reverse>, grid, threads, 0, st, p);
            else launchDependent(decayedRecurrent<T, 128, Reverse>, grid, threads, 0, st, p);
        };
        if (p.reverse) run(std::true_type{});
        else run(std::false_type{});
        afterLaunch("decayedRecurrent");
    });
}

}  // namespace decayed
}  // namespace rxmet
