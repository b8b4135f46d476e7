// Linear attention with a decay for each head over chunks of 128 tokens, on tcgen05.
//
// With l the decay, S the state in front of a chunk of n tokens and i, j tokens of it (forward in time; the reverse pass mirrors the exponents):
//   O = scale (l^(i+1) Q S + ((Q K') . [i >= j] l^(i-j)) V)          S <- l^n S + K'^T diag(l^(n-1-j)) V
// Exponents are differences of places in a chunk and never negative, so that no power overflows.  A CTA walks over the chunks of one head and of 64 columns of V, warps by role:
//   copies     Q, K and V of the next chunks as TMA boxes with a 128-byte swizzle
//   products   one thread issues P = Q K', KV = (weighted K)' V, O1 = Q S and O2 = P V
//   scores     eight warps: P from tensor memory, times the decays, back as the A operand of the last product; then O1 and O2 to the output tile, which TMA stores
//   state      eight warps: weighted K, transposed, into tensor memory as the A operand of KV; the state itself, 32 bits, stays in their registers
//
// Roundings.  Operands of tensor cores have the type of the inputs: P times the decays and S are rounded to it once, next to the rounding of the output.  The state is never
// rebuilt from rounded values: the weighted K goes in as the sum of three bfloat16 or two half terms, which leaves 2^-24.  half has a short range: its rows of P and its S are scaled by
// powers of two to the top of it, and the second term of the weighted K is scaled by 2^11 and summed apart.
#include "decayed_attention.h"
#include "dependent_launch.cuh"
#include "element_types.cuh"
#include "umma_tiles.cuh"

namespace rxmet {
namespace decayed {
namespace {

using namespace ummatiles;

constexpr int kC = kChunkTokens;
constexpr int kCols = 64;              // columns of V a CTA takes
constexpr int kScoreWarps = 8, kStateWarps = 8, kCopyWarp = 16, kProductWarp = 17;
constexpr int kThreads = 32 * 18;
constexpr uint32_t kTile = kC * 128;   // 128 rows of 64 elements
constexpr uint32_t kShared = 229888;   // with up to 2.5 KB of static arrays all of an SM, as the tensor memory
// columns of tensor memory
constexpr uint32_t kP = 0, kO1 = 128, kO2 = 192, kKV = 256, kWeightedK = 320, kKVLow = 448;

struct Segments {
    int count, chunks;   // segments of time, chunks of a segment
    float *states;       // [batch][heads][count][key][value]: ends of the segments on their own, then their beginnings
};

// Place of a segment in the order of the pass, its chunks and tokens.
struct Span {
    int total, first, chunks;   // chunks of the row; the segment's, in the order of the pass
    __host__ __device__ Span(int length, int segment, int segmentChunks) {
        total = (length + kC - 1) / kC;
        first = segment * segmentChunks;
        chunks = total - first < segmentChunks ? total - first : segmentChunks;
        if (chunks < 0) chunks = 0;
    }
    __host__ __device__ int chunkAt(int u, bool reverse) const { return reverse ? total - 1 - first - u : first + u; }
    __host__ __device__ int tokens(int length, bool reverse) const {
        if (chunks == 0) return 0;
        const int a = chunkAt(0, reverse), b = chunkAt(chunks - 1, reverse), low = a < b ? a : b, high = a < b ? b : a;
        const int end = (high + 1) * kC < length ? (high + 1) * kC : length;
        return end - low * kC;
    }
};

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return packBf16(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return make_float2(bf16Lo(v), bf16Hi(v)); }
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }

// The power of two that brings magnitudes up to `most` below 2^15; 1 where there is nothing to scale.
__device__ __forceinline__ float toTopOfHalf(float most) {
    if (!(most > 0.f) || isinf(most)) return 1.f;
    const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;   // floor(log2), -127 below the normal range
    const int up = min(14 - e, 100);
    return __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
}

// DK: elements of a key that the tiles hold, 64 or 128.  StateOnly: nothing but the state at the end of the segment.
template <class T, int DK, bool StateOnly>
__global__ void __launch_bounds__(kThreads, 1)
    decayedChunks(const __grid_constant__ Pass p, const __grid_constant__ CUtensorMap qMap, const __grid_constant__ CUtensorMap kMap, const __grid_constant__ CUtensorMap vMap,
                  const __grid_constant__ CUtensorMap outMap, const bool storeBoxes, const Segments segments, const int terms, int *status) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kHalves = DK / 64;
    constexpr uint32_t kStageBytes = (2 * kHalves + 1) * kTile;
    constexpr int kStages = DK == 64 ? 3 : 2;
    constexpr uint32_t kSBytes = DK * 128;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(16) float powers[kC + 4], columnPowers[32], weights[kC];   // l^n; l^(31 - j) or l^j of a block's columns; of the tokens in the new state
    __shared__ float rowPeaks[2][kC], statePeaks[kStateWarps], stateScale[2];
    __shared__ __align__(8) uint64_t full[kStages], freed[kStages], pFull, pReady, aReady, kvFull, sReady, sFree, oFull, oFree;
    __shared__ uint32_t tmemSlot;
    __shared__ int failed;

    const int warp = warpIndex(), lane = threadIdx.x & 31, tid = threadIdx.x;
    const int slices = gridDim.x / segments.count, slice = blockIdx.x % slices, segment = blockIdx.x / slices, h = blockIdx.y, b = blockIdx.z;
    const uint32_t tiles = (smemAddr(raw) + 1023u) & ~1023u;
    const uint32_t sTile = tiles + kStages * kStageBytes, oTile = sTile + kSBytes;
    const bool reverse = p.reverse;

    waitForPredecessor();
    const int length = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
    const Span span(length, segment, segments.chunks);
    const int count = span.chunks;
    auto tokensOf = [&](int chunk) { return min(kC, length - chunk * kC); };

    if (tid == 0) {
        failed = 0;
        for (int i = 0; i < kStages; ++i) { cluster::initBarrier(&full[i], 1); cluster::initBarrier(&freed[i], 1); }
        for (uint64_t *bar : {&pFull, &kvFull, &sFree, &oFull}) cluster::initBarrier(bar, 1);
        for (uint64_t *bar : {&pReady, &oFree}) cluster::initBarrier(bar, kScoreWarps);
        for (uint64_t *bar : {&aReady, &sReady}) cluster::initBarrier(bar, kStateWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid <= kC) {
        const double g = p.logDecay[h];
        powers[tid] = tid == 0 ? 1.f : static_cast<float>(exp(tid * g));
    } else if (tid >= 256 && tid < 288) {
        const int apart = reverse ? tid - 256 : 287 - tid;
        columnPowers[tid - 256] = apart == 0 ? 1.f : static_cast<float>(exp(apart * static_cast<double>(p.logDecay[h])));
    }
    if (warp == kProductWarp) allocTmem<1>(smemAddr(&tmemSlot), 512);
    fenceBefore();
    __syncthreads();
    fenceAfter();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmemSlot, 0);
    letDependentsStart();

    bool alive = true;
    auto wait = [&](uint64_t &bar, uint32_t parity) {
        if (alive) alive = __all_sync(0xffffffffu, waitSuspended(smemAddr(&bar), parity));
    };
    auto arriveWarp = [&](uint64_t &bar) {
        __syncwarp();
        if (lane == 0) arrive(smemAddr(&bar));
    };

    if (warp == kCopyWarp) {
        Turn turn;
        for (int u = 0; u < count; ++u, turn.step(kStages)) {
            if (turn.again) wait(freed[turn.at], turn.parity ^ 1u);
            if (alive && electOne()) {
                const uint32_t bar = smemAddr(&full[turn.at]), to = tiles + turn.at * kStageBytes;
                const int t = span.chunkAt(u, reverse) * kC;
                cluster::arriveExpect(bar, StateOnly ? (kHalves + 1) * kTile : kStageBytes);
                if (!StateOnly)
                    for (int i = 0; i < kHalves; ++i) copyTile4(to + i * kTile, &qMap, 64 * i, h / (p.heads / p.q.heads), t, b, bar);
                for (int i = 0; i < kHalves; ++i) copyTile4(to + (kHalves + i) * kTile, &kMap, 64 * i, h / (p.heads / p.k.heads), t, b, bar);
                copyTile4(to + 2 * kHalves * kTile, &vMap, slice * kCols, h / (p.heads / p.v.heads), t, b, bar);
            }
            __syncwarp();
        }
        // nothing is left in flight: the products of the last use of each stage are complete
        for (int i = 0; i < kStages; ++i, turn.step(kStages))
            if (turn.again) waitSuspended(smemAddr(&freed[turn.at]), turn.parity ^ 1u);
    } else if (warp == kProductWarp) {
        constexpr uint32_t kScores = halves(!kHalf, kC, false), kOthers = halves(!kHalf, kCols, true);
        Turn turn;
        for (int u = 0; u < count; ++u, turn.step(kStages)) {
            const uint32_t at = tiles + turn.at * kStageBytes, parity = u & 1;
            const uint64_t q = swizzledDescriptor(at), k = swizzledDescriptor(at + kHalves * kTile), v = swizzledDescriptor(at + 2 * kHalves * kTile), s = swizzledDescriptor(sTile);
            wait(full[turn.at], turn.parity);
            if (!StateOnly) {
                if (u > 0) wait(oFull, parity ^ 1u);   // the last product has read P
                if (alive && electOne()) {
                    fenceAfter();
#pragma unroll
                    for (int i = 0; i < 4 * kHalves; ++i) {
                        const uint64_t step = (i / 4) * (kTile >> 4) + (i % 4) * 2;
                        product(tmem + kP, q + step, k + step, kScores, i > 0);
                    }
                    commitTo(smemAddr(&pFull));
                }
                __syncwarp();
            }
            wait(aReady, parity);
            if (alive && electOne()) {
                fenceAfter();
                for (int term = terms - 1; term >= 0; --term) {
                    const bool low = kHalf && term > 0;
#pragma unroll
                    for (int i = 0; i < kC / 16; ++i)
                        productTmem(tmem + (low ? kKVLow : kKV), tmem + kWeightedK + term * 64 + i * 8, v + i * 128, kOthers, i > 0 || (!kHalf && term < terms - 1));
                }
                commitTo(smemAddr(&kvFull));
                if (StateOnly) commitTo(smemAddr(&freed[turn.at]));
            }
            __syncwarp();
            if (!StateOnly) {
                wait(sReady, parity);
                if (u > 0) wait(oFree, parity ^ 1u);
                if (alive && electOne()) {
                    fenceAfter();
#pragma unroll
                    for (int i = 0; i < DK / 16; ++i) product(tmem + kO1, q + (i / 4) * (kTile >> 4) + (i % 4) * 2, s + i * 128, kOthers, i > 0);
                    commitTo(smemAddr(&sFree));
                }
                __syncwarp();
                wait(pReady, parity);
                if (alive && electOne()) {
                    fenceAfter();
#pragma unroll
                    for (int i = 0; i < kC / 16; ++i) productTmem(tmem + kO2, tmem + kP + i * 8, v + i * 128, kOthers, i > 0);
                    commitTo(smemAddr(&oFull));
                    commitTo(smemAddr(&freed[turn.at]));
                }
                __syncwarp();
            }
        }
    } else if (warp < kScoreWarps) {
        if (!StateOnly) {
            const int quarter = warp & 3, half = warp >> 2, i = 32 * quarter + lane;   // the thread's token; of each block of 32 columns it takes 16
            const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
            for (int u = 0; u < count; ++u) {
                const uint32_t parity = u & 1;
                const int chunk = span.chunkAt(u, reverse), n = tokensOf(chunk);
                wait(pFull, parity);
                fenceAfter();
                // bfloat16 is packed block by block; half waits for the largest score of the row
                constexpr int kKept = kHalf ? 4 : 1;
                float scores[kKept][16];
                uint32_t words[4][8] = {};
                float most = 0.f;
                auto empty = [&](int block) { return reverse ? block < quarter : block > quarter; };
#pragma unroll
                for (int block = 0; block < 4; ++block) {
                    if (empty(block)) continue;
                    float(&mine)[16] = scores[kHalf ? block : 0];
                    uint32_t r[16];
                    loadTmem16(lanes + kP + block * 32 + half * 16, r);
                    loadsDone();
                    const int first = block * 32 + half * 16;
                    if (block == quarter) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int apart = reverse ? first + j - i : i - first - j;
                            const bool in = apart >= 0 && (!reverse || first + j < n);
                            mine[j] = in ? __uint_as_float(r[j]) * powers[max(apart, 0)] * p.outScale : 0.f;
                        }
                    } else {
                        const float row = p.outScale * powers[reverse ? block * 32 - i : i - block * 32 - 31];
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 c = *reinterpret_cast<const float4 *>(&columnPowers[half * 16 + j]);
                            const float cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) mine[j + e] = __uint_as_float(r[j + e]) * cs[e] * row;
                        }
                        if (reverse && n < kC) {   // tokens behind the row's end may hold anything
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (first + j >= n) mine[j] = 0.f;
                        }
                    }
                    if constexpr (kHalf) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) most = fmaxf(most, fabsf(mine[j]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) words[block][j] = pack2<T>(mine[2 * j], mine[2 * j + 1]);
                    }
                }
                float back = 1.f;
                if (kHalf) rowPeaks[half][i] = most;
                groupBarrier(4 + quarter, 64);   // both warps of these lanes have read P, which is written over
                if constexpr (kHalf) {
                    const float up = toTopOfHalf(fmaxf(most, rowPeaks[half ^ 1][i]));
                    back = 1.f / up;
#pragma unroll
                    for (int block = 0; block < 4; ++block)
                        if (!empty(block))
#pragma unroll
                            for (int j = 0; j < 8; ++j) words[block][j] = pack2<T>(scores[block][2 * j] * up, scores[block][2 * j + 1] * up);
                }
#pragma unroll
                for (int block = 0; block < 4; ++block) storeTmem8(lanes + kP + block * 16 + half * 8, words[block]);
                tmemStoresDone();
                fenceBefore();
                arriveWarp(pReady);

                wait(oFull, parity);
                fenceAfter();
                const bool live = i < n;
                const float inter = live ? p.outScale * powers[reverse ? n - 1 - i : i + 1] * (kHalf ? stateScale[parity] : 1.f) : 0.f;
                float out[32];
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    uint32_t o1[16], o2[16];
                    loadTmem16(lanes + kO1 + half * 32 + part * 16, o1);
                    loadTmem16(lanes + kO2 + half * 32 + part * 16, o2);
                    loadsDone();
#pragma unroll
                    for (int j = 0; j < 16; ++j) out[part * 16 + j] = live ? fmaf(__uint_as_float(o1[j]), inter, __uint_as_float(o2[j]) * back) : 0.f;
                }
                fenceBefore();
                arriveWarp(oFree);
                if (storeBoxes) {
                    if (tid == 0) storesRead();   // the tile's last copy
                    groupBarrier(1, 32 * kScoreWarps);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = pack2<T>(out[8 * c + 2 * j], out[8 * c + 2 * j + 1]);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(oTile + i * 128 + (((half * 4 + c) ^ (i & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                    }
                    fenceAsyncProxy();
                    groupBarrier(1, 32 * kScoreWarps);
                    if (tid == 0 && alive) storeTile4(&outMap, oTile, slice * kCols, h, chunk * kC, b);
                } else if (p.out && chunk * kC + i < p.tokens && alive) {
                    const int col = slice * kCols + half * 32;
                    const size_t at = ((static_cast<size_t>(b) * p.tokens + chunk * kC + i) * p.heads + h) * p.value + col;
                    if (p.outFloat && p.value % 4 == 0) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            if (col + j < p.value) *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at + j) = make_float4(out[j], out[j + 1], out[j + 2], out[j + 3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (col + j >= p.value) continue;
                            if (p.outFloat) static_cast<float *>(p.out)[at + j] = out[j];
                            else static_cast<T *>(p.out)[at + j] = fromFloat<T>(out[j]);
                        }
                    }
                }
            }
            if (storeBoxes && tid == 0) storesDone();
        }
    } else {
        const int quarter = warp & 3, half = (warp - kScoreWarps) >> 2, d = 32 * quarter + lane;   // the thread's row of the state, and which half of its columns and of the tokens
        const bool rows = 32 * quarter < DK;                                                     // warps beyond the keys have none
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
        const int stid = tid - 32 * kScoreWarps;
        const size_t head = static_cast<size_t>(b) * p.heads + h, stateSize = static_cast<size_t>(p.key) * p.value;
        const int col = slice * kCols + half * 32;
        float s[32];
        const float *in = segments.count > 1 ? (StateOnly ? nullptr : segments.states + (head * segments.count + segment) * stateSize) : p.stateIn ? p.stateIn + head * stateSize : nullptr;
        const int inRow = segments.count > 1 ? p.value : p.stateRow, inCol = segments.count > 1 ? 1 : p.stateCol;
        const float inScale = segments.count > 1 ? 1.f : p.inScale;
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = in && d < p.key && col + j < p.value ? inScale * in[static_cast<size_t>(d) * inRow + static_cast<size_t>(col + j) * inCol] : 0.f;

        auto publish = [&](int u) {   // the state in front of chunk u, as the B operand of O1
            float up = 1.f;
            if constexpr (kHalf) {
                float most = 0.f;
#pragma unroll
                for (int j = 0; j < 32; ++j) most = fmaxf(most, fabsf(s[j]));
                const uint32_t peak = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
                if (lane == 0) statePeaks[stid >> 5] = __uint_as_float(peak);
                groupBarrier(2, 32 * kStateWarps);
                most = 0.f;
#pragma unroll
                for (int w = 0; w < kStateWarps; ++w) most = fmaxf(most, statePeaks[w]);
                up = toTopOfHalf(most);
                if (stid == 0) stateScale[u & 1] = 1.f / up;
                groupBarrier(2, 32 * kStateWarps);
            }
            if (rows) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = pack2<T>(s[8 * c + 2 * j] * up, s[8 * c + 2 * j + 1] * up);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sTile + d * 128 + (((half * 4 + c) ^ (d & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                }
                fenceAsyncProxy();
            }
            arriveWarp(sReady);
        };
        if (!StateOnly && count > 0) publish(0);

        // byte of element d in each of eight rows of a tile of K
        const uint32_t element = (d & 63) * 2, kHalfTile = (d >> 6) * kTile;
        Turn turn;
        int weighted = -1;   // tokens that `weights` is for
        for (int u = 0; u < count; ++u, turn.step(kStages)) {
            const uint32_t parity = u & 1, at = tiles + turn.at * kStageBytes;
            const int chunk = span.chunkAt(u, reverse), n = tokensOf(chunk);
            if (weighted != n) {
                groupBarrier(2, 32 * kStateWarps);
                if (stid < kC) weights[stid] = stid < n ? powers[reverse ? stid + 1 : n - 1 - stid] : 0.f;
                groupBarrier(2, 32 * kStateWarps);
                weighted = n;
            }
            wait(full[turn.at], turn.parity);
            if (n < kC && chunk * kC + n < p.tokens) {   // V behind the row's end may hold anything, and zero times that is not zero
                for (int i = n * 8 + stid; i < kC * 8; i += 32 * kStateWarps)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + 2 * kHalves * kTile + i * 16), "r"(0u) : "memory");
                fenceAsyncProxy();
            }
            if (rows) {
                const uint32_t keys = at + kHalves * kTile + kHalfTile;
#pragma unroll 1
                for (int j0 = half * 64; j0 < half * 64 + 64; j0 += 16) {
                    uint32_t hi[8], mid[8], lo[8];
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 w4 = *reinterpret_cast<const float4 *>(&weights[j0 + j]);
                        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t r = (j + e) & 7;   // the place of token j0 + j + e among eight rows
                            uint16_t bits;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(keys + (j0 + j + e) * 128 + (element ^ (r << 4))) : "memory");
                            const T value = *reinterpret_cast<const T *>(&bits);
                            x[e] = n == kC || j0 + j + e < n ? toFloat(value) * w[e] : 0.f;
                        }
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const int word = (j + e) / 2;
                            hi[word] = pack2<T>(x[e], x[e + 1]);
                            float2 back = unpack2<T>(hi[word]);
                            float r0 = x[e] - back.x, r1 = x[e + 1] - back.y;
                            if constexpr (kHalf) {
                                mid[word] = pack2<T>(r0 * 2048.f, r1 * 2048.f);
                                lo[word] = 0u;
                            } else {
                                mid[word] = pack2<T>(r0, r1);
                                back = unpack2<T>(mid[word]);
                                lo[word] = pack2<T>(r0 - back.x, r1 - back.y);
                            }
                        }
                    }
                    const uint32_t to = lanes + kWeightedK + j0 / 2;
                    storeTmem8(to, hi);
                    storeTmem8(to + 64, mid);
                    if (!kHalf && terms > 2) storeTmem8(to + 128, lo);
                }
                tmemStoresDone();
            }
            fenceBefore();
            arriveWarp(aReady);

            wait(kvFull, parity);
            fenceAfter();
            const float keep = powers[n];
            if (rows) {
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    uint32_t r[16];
                    loadTmem16(lanes + kKV + half * 32 + part * 16, r);
                    if constexpr (kHalf) {
                        uint32_t low[16];
                        loadTmem16(lanes + kKVLow + half * 32 + part * 16, low);
                        loadsDone();
#pragma unroll
                        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(fmaf(__uint_as_float(low[j]), 1.f / 2048, __uint_as_float(r[j])));
                    } else {
                        loadsDone();
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[part * 16 + j] = fmaf(s[part * 16 + j], keep, __uint_as_float(r[j]));
                }
            }
            if (!StateOnly && u + 1 < count) {
                wait(sFree, parity);
                publish(u + 1);
            }
        }
        float *last = StateOnly ? segments.states + (head * segments.count + segment) * stateSize : segments.count > 1 || !p.stateOut ? nullptr : p.stateOut + head * stateSize;
        if (last && alive) {
            const int outRow = StateOnly ? p.value : p.stateRow, outCol = StateOnly ? 1 : p.stateCol;
            const float scale = StateOnly ? 1.f : p.finalScale;
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (d < p.key && col + j < p.value) last[static_cast<size_t>(d) * outRow + static_cast<size_t>(col + j) * outCol] = s[j] * scale;
        }
    }
    if (!alive && lane == 0) failed = 1;
    if (!StateOnly && p.out) {   // tokens behind the last chunk, of those that lie in this segment's stretch of time
        const int from = max(span.total, segment * segments.chunks) * kC, to = min(p.tokens, (segment + 1) * segments.chunks * kC);
        const int width = min(kCols, p.value - slice * kCols);
        for (int64_t e = tid; e < static_cast<int64_t>(max(0, to - from)) * width; e += kThreads) {
            const size_t at = ((static_cast<size_t>(b) * p.tokens + from + e / width) * p.heads + h) * p.value + slice * kCols + e % width;
            if (p.outFloat) static_cast<float *>(p.out)[at] = 0.f;
            else static_cast<T *>(p.out)[at] = fromFloat<T>(0.f);
        }
    }
    fenceBefore();
    __syncthreads();
    if (warp == kProductWarp) freeTmem<1>(tmem, 512);
    if (tid == 0 && failed) atomicExch(status, 1);
}

// From the ends of the segments on their own to their beginnings: one thread for each element of a state, segment after segment.
__global__ void __launch_bounds__(256) joinSegments(const __grid_constant__ Pass p, const Segments segments) {
    const int h = blockIdx.y, b = blockIdx.z, size = p.key * p.value, e = blockIdx.x * 256 + threadIdx.x;
    waitForPredecessor();
    letDependentsStart();
    if (e >= size) return;
    const int length = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
    const double g = p.logDecay[h];
    const size_t head = static_cast<size_t>(b) * p.heads + h, at = head * size + static_cast<size_t>(e / p.value) * p.stateRow + static_cast<size_t>(e % p.value) * p.stateCol;
    float state = p.stateIn ? p.inScale * p.stateIn[at] : 0.f;
    for (int segment = 0; segment < segments.count; ++segment) {
        float *own = segments.states + (head * segments.count + segment) * size + e;
        const int tokens = Span(length, segment, segments.chunks).tokens(length, p.reverse);
        const float added = tokens > 0 ? *own : 0.f;
        *own = state;
        if (tokens > 0) state = fmaf(state, static_cast<float>(exp(tokens * g)), added);
    }
    if (p.stateOut) p.stateOut[at] = state * p.finalScale;
}

// [batch][tokens][heads][width] with the strides of `t`: boxes of 128 tokens and 64 elements of a head.
CUtensorMap tokenMap(const rxmet_head_tensor &t, int batch, int tokens, int width, bool bf16, bool &ok) {
    CUtensorMap map;
    auto stride = [](int64_t elements, int count) { return static_cast<cuuint64_t>(count > 1 ? elements * 2 : 16); };   // of one element it does not matter
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(t.heads), static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(batch)};
    const cuuint64_t strides[3] = {stride(t.stride_h, t.heads), stride(t.stride_t, tokens), stride(t.stride_b, batch)};
    const cuuint32_t box[4] = {64, 1, kC, 1}, steps[4] = {1, 1, 1, 1};
    ok = ok && encodeTiled()(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(t.data), dims, strides, box, steps,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    return map;
}

bool copies(const rxmet_head_tensor &t, int batch, int tokens) {
    auto fits = [](int64_t stride, int count) { return count == 1 || (stride > 0 && stride % 8 == 0 && stride < (int64_t{1} << 38)); };
    return alignedTo(t.data, 16) && fits(t.stride_h, t.heads) && fits(t.stride_t, tokens) && fits(t.stride_b, batch);
}

}  // namespace

ChunkPlan planChunks(const Pass &p, int type) {
    ChunkPlan plan{type != RXMET_TYPE_F32 && p.tokens >= 32 && encodeTiled() != nullptr, 1, (p.tokens + kC - 1) / kC};
    const int64_t ctas = static_cast<int64_t>((p.value + kCols - 1) / kCols) * p.heads * p.batch;
    const int chunks = plan.segmentChunks, most = static_cast<int>(std::min<int64_t>(chunks / 2, currentDevice().sms / std::max<int64_t>(1, ctas)));
    if (plan.taken && most >= 2) {
        plan.segmentChunks = (chunks + most - 1) / most;
        plan.segments = (chunks + plan.segmentChunks - 1) / plan.segmentChunks;
    }
    return plan;
}

bool chunksCanCopy(const Pass &p) { return copies(p.q, p.batch, p.tokens) && copies(p.k, p.batch, p.tokens) && copies(p.v, p.batch, p.tokens); }

void launchChunks(const Pass &p, int type, const ChunkPlan &plan, float *states, cudaStream_t st) {
    const bool bf16 = type == RXMET_TYPE_BF16;
    bool ok = true;
    bindContext();
    const CUtensorMap q = tokenMap(p.q, p.batch, p.tokens, p.key, bf16, ok), k = tokenMap(p.k, p.batch, p.tokens, p.key, bf16, ok), v = tokenMap(p.v, p.batch, p.tokens, p.value, bf16, ok);
    const bool storeBoxes = p.out && !p.outFloat && p.value % 8 == 0 && alignedTo(p.out, 16);
    CUtensorMap out = q;
    if (storeBoxes) {
        const int64_t row = static_cast<int64_t>(p.heads) * p.value;
        out = tokenMap({p.out, row * p.tokens, row, p.value, p.heads}, p.batch, p.tokens, p.value, bf16, ok);
    }
    if (!ok) fail(RXMET_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    const Segments segments{plan.segments, plan.segmentChunks, states};
    const dim3 grid((p.value + kCols - 1) / kCols * plan.segments, p.heads, p.batch);
    auto run = [&](auto kernel, const char *name, int terms) {
        ensureDynamicSmem(reinterpret_cast<const void *>(kernel), kShared);
        {
            KernelTimer timer__(name, st);
            launchDependent(kernel, grid, kThreads, kShared, st, p, q, k, v, out, storeBoxes, segments, terms, waitStatus());
        }
        afterLaunch(name);
    };
    // Three bfloat16 terms of the weighted K where the state is an output; two, 2^-17, where it only feeds products that round it to 2^-9.
    const int terms = bf16 && p.stateOut ? 3 : 2;
    auto both = [&](auto t, auto dk) {
        using T = decltype(t);
        constexpr int DK = decltype(dk)::value;
        if (plan.segments > 1) {
            run(decayedChunks<T, DK, true>, "decayedChunksState", terms);
            {
                KernelTimer timer__("joinSegments", st);
                launchDependent(joinSegments, dim3((p.key * p.value + 255) / 256, p.heads, p.batch), 256, 0, st, p, segments);
            }
            afterLaunch("joinSegments");
        }
        if (p.out || plan.segments == 1) run(decayedChunks<T, DK, false>, "decayedChunks", plan.segments > 1 ? 2 : terms);
    };
    auto withKeys = [&](auto t) {
        if (p.key <= 64) both(t, std::integral_constant<int, 64>{});
        else both(t, std::integral_constant<int, 128>{});
    };
    if (bf16) withKeys(__nv_bfloat16{});
    else withKeys(__half{});
}

}  // namespace decayed
}  // namespace rxmet
