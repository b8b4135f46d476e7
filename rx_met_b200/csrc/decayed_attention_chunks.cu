// Linear attention with a decay for each head over chunks of 128 tokens, on tcgen05.
//
// With l the decay, S the state in front of a chunk of n tokens and i, j tokens of it (forward in time; the reverse pass mirrors the exponents):
//   O = scale (l^(i+1) Q S + ((Q K') . [i >= j] l^(i-j)) V)          S <- l^n S + K'^T diag(l^(n-1-j)) V
// Exponents are differences of places in a chunk and never negative, so that no power overflows.  A CTA walks over the chunks of one head and of 64 columns of V, warps by role:
//   copies     Q, K and V of the next chunks as TMA boxes with a 128-byte swizzle
//   products   two threads issue KV = K'^T (weighted V) and O1 = Q S, and P = Q K' and O2 = P V; P has two buffers,
//              so that the next product may run under a chunk's scores
//   scores     eight warps: P from tensor memory, times the decays, back as the A operand of the last product
//   outputs    four warps: O1 and O2 to memory, 32 bytes a thread and store
//   state      eight warps: weighted V for the products; the state itself, 32 bits, stays in their registers
//
// P is zero in front of a token, and zero times an infinity or a NaN of V is not: such values, which leave a NaN in the weighted V, are taken out of the V of the last product once the
// weighted V has them, and outputs says NaN for their column from their token on.
//
// Roundings.  Operands of tensor cores have the type of the inputs: P times the decays and S are rounded to it once, next to the rounding of the output.  The state is never
// rebuilt from rounded values: the weighted V goes in as the sum of three bfloat16 terms, which leave 2^-24, or two of half,
// 2^-22.  half has a short range: its rows of P, its S and the weighted V of a chunk are scaled by
// powers of two to the top of it, the second term of the weighted V by 2^11 more (unscaled, values of 1e-6 left 2^-16; 1 x 16384 tokens of 8 heads of 64 45 -> 46.5 us).  The two larger terms lie side by side as 128 columns of one product, which reads
// K once for both.  All chunks have the third term: later ones may add little, so that what an early one leaves in the state is all of it (8 x 4096 tokens of 16 heads of 128: 163 us, 152 with
// the third term of the last chunks alone, whose states were off by 2^-18.6 there).
//
// Bound: the chain of a chunk (terms of V, their product, the state, its rounding, Q S), about 3400 cycles with 64 keys and 4300 with 128 of which the tensor cores work two fifths, the issue slots half; and
// one CTA an SM.  8 x 4096 tokens of 16 heads: 163 us with 128 elements a head (3.3 TB/s, two rounds of CTAs), 66 with 64 (4.1 TB/s); half, whose scales take a turn more over scores,
// state and V, 175 and 85.
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
constexpr int kScoreWarps = 8, kOutputWarps = 4, kStateWarps = 8;
constexpr int kFirstOutput = kScoreWarps, kFirstState = kFirstOutput + kOutputWarps, kCopyWarp = kFirstState + kStateWarps, kStateProducts = kCopyWarp + 1, kScoreProducts = kStateProducts + 1;
constexpr int kThreads = 32 * 24;   // the last warp has no work: registers are dealt to groups of four warps
constexpr uint32_t kTile = kC * 128;   // 128 rows of 64 elements
constexpr uint32_t kShared = 232448;   // all of an SM, as the tensor memory
// columns of tensor memory: two buffers of P, then the others; KV is the larger term and then the others
constexpr uint32_t kP = 0, kO1 = 256, kO2 = 320, kKV = 384;
enum Barrier { kStateMeets = 1, kLanesMeet };   // named barriers; the last takes four

// A block starts with 80 registers a thread, 1920 for the lanes of its 24 warps in the same place.  Scores give up 8 (8 warps, 576), outputs 24 (4 warps, 224), copies and products 40 (4
// warps, 160), and the state takes 120 (8 warps, 960): 1920.  With 80 the state would be spilled (advance() 420 -> 1700 cycles), with 104 its third terms.
template <int REGISTERS>
__device__ __forceinline__ void giveRegisters() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGISTERS)); }
template <int REGISTERS>
__device__ __forceinline__ void takeRegisters() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGISTERS)); }

// Shared memory in groups of 16 bytes.
__device__ __forceinline__ void loadShared(uint32_t at, uint32_t (&v)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void storeShared(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Two neighbours of a 16-bit type: NaN where the value is not finite, else what was there.
template <class T>
__device__ __forceinline__ void addZeroTimes(uint32_t &sum, uint32_t value) {
    if constexpr (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(value), "r"(0u));
    else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(value), "r"(0u));
}
// Orders tokens of the chunks of a pass: a later chunk's keys are larger, and of a chunk's tokens that of the first in the order of the pass.
__device__ __forceinline__ uint32_t badKey(int u, int token, bool reverse) { return static_cast<uint32_t>(u + 1) << 8 | static_cast<uint32_t>(reverse ? token + 1 : 255 - token); }
// Takes what is not finite out of 32 values of V, those of a token in the four pieces of 16 bytes from `piece` on, and keeps where.
template <class T>
__device__ __forceinline__ void clean(uint32_t row, uint32_t swizzle, uint32_t piece, uint32_t *badFrom, uint32_t key) {
#pragma unroll 1
    for (uint32_t i = 0; i < 16; ++i) {
        const uint32_t at = row + (((piece + (i >> 2)) ^ swizzle) << 4) + (i & 3) * 4;
        uint32_t w, kept;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
        kept = w;
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j)
            if ((w >> (16 * j) & 0x7fffu) >= (std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u)) {
                kept &= j ? 0xffffu : 0xffff0000u;
                atomicMax(&badFrom[(piece + (i >> 2)) * 8 + (i & 3) * 2 + j], key);
            }
        if (kept != w) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(kept) : "memory");
    }
}

constexpr int kMaxSegments = 160;   // no more than SMs
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

// The power of two that brings magnitudes up to one with the exponent bits `exponent` below 2^15; 1 where there is nothing to scale.
__device__ __forceinline__ uint32_t exponentBits(float most) { return __float_as_uint(most) >> 23; }
__device__ __forceinline__ float toTopOfHalf(uint32_t exponent) {
    if (exponent == 0 || exponent == 255) return 1.f;   // none that a half could show; infinite
    return __uint_as_float(static_cast<uint32_t>(127 + min(14 + 127 - static_cast<int>(exponent), 100)) << 23);
}

// What a CTA keeps in shared memory beside the tiles.
struct Small {
    float powers[kC + 4], scaledPowers[32], columnPowers[32];   // l^n; scale l^n; scale l^(31 - j) or scale l^j of a block's columns
    float statePeaks[2][kStateWarps], valuePeaks[2][kStateWarps], stateScale[2];   // of two chunks in turn, so that the warps meet once a chunk
    uint8_t rowPeaks[2][2][kC];               // exponents, of two chunks in turn
    uint8_t rowScale[3][kC];                  // exponents of the powers of two that rows of P were scaled by, for three chunks
    uint32_t badFrom[3][kCols];               // where outputs of a column stop being finite, of three chunks in turn (badKey)
    uint32_t lastBad;                         // the last chunk where they do, counted from 1
    uint64_t fullK[3], fullQ[3], fullV[3], freeK[3], freeQ[3], freeV[3], vRead[3], pFull[2], pReady[2], pFree[2], vReady, kvFull, sReady, sFree, oFull, oFree, productsDone[2];
    uint32_t tmemSlot;
    int failed;
};

// DK: elements of a key that the tiles hold, 64 or 128.  Third: bfloat16 with a third term of the weighted V.  StateOnly: nothing but the state at the end of the segment.  Stores: how outputs leave, by the alignment of their
// rows.
enum class Stores { Elements, Packed, Floats };   // one by one; sixteen of the type of the inputs, or eight in 32 bits, at a time
template <class T, int DK, bool Third, bool StateOnly, Stores How>
__global__ void __launch_bounds__(kThreads, 1)
    decayedChunks(const __grid_constant__ Pass p, const __grid_constant__ CUtensorMap qMap, const __grid_constant__ CUtensorMap kMap, const __grid_constant__ CUtensorMap vMap,
                  const Segments segments, int *status) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kHalves = DK / 64;
    constexpr uint32_t kStageBytes = (2 * kHalves + 1) * kTile;
    constexpr int kStages = DK == 64 ? 3 : 2;
    constexpr uint32_t kSBytes = DK * 128;
    static_assert(kStages * kStageBytes + kSBytes + 3 * kTile + sizeof(Small) <= kShared, "shared memory");
    extern __shared__ __align__(1024) uint8_t raw[];
    const uint32_t tiles = smemAddr(raw), sTile = tiles + kStages * kStageBytes, weightedV = sTile + kSBytes;
    Small &small = *reinterpret_cast<Small *>(raw + kStages * kStageBytes + kSBytes + 3 * kTile);

    const int warp = warpIndex(), lane = threadIdx.x & 31, tid = threadIdx.x;
    const int slices = gridDim.x / segments.count, slice = blockIdx.x % slices, segment = blockIdx.x / slices, h = blockIdx.y, b = blockIdx.z;
    const bool reverse = p.reverse;

    waitForPredecessor();
    const int length = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
    const Span span(length, segment, segments.chunks);
    const int count = span.chunks;
    auto tokensOf = [&](int chunk) { return min(kC, length - chunk * kC); };
    if (tid == 0) {
        small.failed = 0;
        small.lastBad = 0;
        for (int i = 0; i < kStages; ++i)
            for (uint64_t *bar : {&small.fullK[i], &small.fullQ[i], &small.fullV[i], &small.freeV[i]}) cluster::initBarrier(bar, 1);
        constexpr int kUsers = StateOnly ? 1 : 2;   // threads whose products read K and Q, and write O1 and O2
        for (int i = 0; i < kStages; ++i)
            for (uint64_t *bar : {&small.freeK[i], &small.freeQ[i]}) cluster::initBarrier(bar, kUsers);
        cluster::initBarrier(&small.oFull, kUsers);
        for (uint64_t *bar : {&small.pFull[0], &small.pFull[1], &small.pFree[0], &small.pFree[1], &small.kvFull, &small.sFree, &small.productsDone[0], &small.productsDone[1]}) cluster::initBarrier(bar, 1);
        // Barriers for each buffer of P: a chunk's scores may be done before the products have asked for those of the chunk before.
        for (uint64_t *bar : {&small.pReady[0], &small.pReady[1]}) cluster::initBarrier(bar, kScoreWarps);
        // One for each stage: the state may be two chunks ahead of the scores, and a barrier in its phase after next looks like one that is not over.
        for (int i = 0; i < kStages; ++i) cluster::initBarrier(&small.vRead[i], kStateWarps);
        cluster::initBarrier(&small.oFree, kOutputWarps);
        for (uint64_t *bar : {&small.vReady, &small.sReady}) cluster::initBarrier(bar, kStateWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid <= kC) {
        const double g = p.logDecay[h];
        small.powers[tid] = tid == 0 ? 1.f : static_cast<float>(exp(tid * g));
    } else if (tid >= 384 && tid < 384 + 3 * kCols) {
        small.badFrom[0][tid - 384] = 0;
    } else if (tid >= 256 && tid < 320) {
        const int j = tid & 31, apart = tid < 288 || reverse ? j : 31 - j;
        (tid < 288 ? small.scaledPowers : small.columnPowers)[j] = p.outScale * (apart == 0 ? 1.f : static_cast<float>(exp(apart * static_cast<double>(p.logDecay[h]))));
    }
    if (warp == kStateProducts) allocTmem<1>(smemAddr(&small.tmemSlot), 512);
    fenceBefore();
    __syncthreads();
    fenceAfter();
    const uint32_t tmem = __shfl_sync(0xffffffffu, small.tmemSlot, 0);
    letDependentsStart();

    bool alive = true;
    auto wait = [&](uint64_t &bar, uint32_t parity) {
        if (alive) alive = __all_sync(0xffffffffu, waitSuspended(smemAddr(&bar), parity));
    };
    auto arriveWarp = [&](uint64_t &bar) {
        __syncwarp();
        if (lane == 0) arrive(smemAddr(&bar));
    };

    if (warp >= kCopyWarp) {
        // The test stands alone in front of the three roles: only so does the compiler see whose registers these are.
        giveRegisters<40>();
        if (warp == kCopyWarp) {
            Turn turn;
            for (int u = 0; u < count; ++u, turn.step(kStages)) {
                // each as soon as its last use is over, in the order in which that is
                const uint32_t to = tiles + turn.at * kStageBytes;
                const int t = span.chunkAt(u, reverse) * kC;
                auto fetch = [&](uint64_t &full, uint64_t &free, const CUtensorMap &map, uint32_t place, int boxes, int x, int head) {
                    if (turn.again) wait(free, turn.parity ^ 1u);
                    if (alive && electOne()) {
                        cluster::arriveExpect(smemAddr(&full), boxes * kTile);
                        for (int i = 0; i < boxes; ++i) copyTile4(to + place + i * kTile, &map, x + 64 * i, head, t, b, smemAddr(&full));
                    }
                    __syncwarp();
                };
                fetch(small.fullK[turn.at], small.freeK[turn.at], kMap, kHalves * kTile, kHalves, 0, h / (p.heads / p.k.heads));
                if (!StateOnly) fetch(small.fullQ[turn.at], small.freeQ[turn.at], qMap, 0, kHalves, 0, h / (p.heads / p.q.heads));
                fetch(small.fullV[turn.at], small.freeV[turn.at], vMap, 2 * kHalves * kTile, 1, slice * kCols, h / (p.heads / p.v.heads));
            }
            // nothing is left in flight: the last use of each stage is over
            for (int i = 0; i < kStages; ++i, turn.step(kStages))
                if (turn.again) {
                    waitSuspended(smemAddr(&small.freeK[turn.at]), turn.parity ^ 1u);
                    if (!StateOnly) waitSuspended(smemAddr(&small.freeQ[turn.at]), turn.parity ^ 1u);
                    waitSuspended(smemAddr(&small.freeV[turn.at]), turn.parity ^ 1u);
                }
        } else if (warp <= kScoreProducts) {
            // Two threads issue the products, those of the state and those of the scores: one alone came to 4200 cycles a chunk, of which the tensor cores work 1300.  They poll, because a
            // vote of the warp after each wait costs 150 cycles.
            constexpr uint32_t kScores = halves(!kHalf, kC, false, false), kOutputs = halves(!kHalf, kCols, false, true);
            constexpr uint32_t kBothTerms = halves(!kHalf, 2 * kCols, true, true), kThirdTerm = halves(!kHalf, kCols, true, true);
            auto poll = [&](uint64_t &bar, uint32_t parity) {
                if (alive) alive = waitPhase(smemAddr(&bar), parity);
                fenceAfter();
            };
            if (warp == kStateProducts) {
                if (electOne()) {
                    Turn turn;
                    const uint64_t weighted = swizzledDescriptor(weightedV, kTile), third = swizzledDescriptor(weightedV + 2 * kTile), s = swizzledDescriptor(sTile);
                    for (int u = 0; u < count; ++u, turn.step(kStages)) {
                        const uint32_t at = tiles + turn.at * kStageBytes, parity = u & 1, kv = tmem + kKV;
                        const uint64_t q = swizzledDescriptor(at), k = swizzledDescriptor(at + kHalves * kTile, kHalves == 2 ? kTile : 0);   // 64 keys: a stride of 0 lays them down twice, in rows 0 and 64 of KV
                        poll(small.fullK[turn.at], turn.parity);
                        poll(small.vReady, parity);
#pragma unroll 2
                        for (int i = 0; i < kC / 16; ++i) product(kv, k + i * 128, weighted + i * 128, kBothTerms, i > 0);
                        if (Third) {
#pragma unroll 2
                            for (int i = 0; i < kC / 16; ++i) product(kv + kCols, k + i * 128, third + i * 128, kThirdTerm, 1);
                        }
                        commitTo(smemAddr(&small.kvFull));
                        commitTo(smemAddr(&small.freeK[turn.at]));
                        if (StateOnly) {
                            commitTo(smemAddr(&small.freeV[turn.at]));
                            continue;
                        }
                        poll(small.fullQ[turn.at], turn.parity);
                        poll(small.sReady, parity);
                        if (u > 0) poll(small.oFree, parity ^ 1u);
#pragma unroll 2
                        for (int i = 0; i < DK / 16; ++i) product(tmem + kO1, q + (i / 4) * (kTile >> 4) + (i % 4) * 2, s + i * 128, kOutputs, i > 0);
                        commitTo(smemAddr(&small.sFree));
                        commitTo(smemAddr(&small.freeQ[turn.at]));
                        commitTo(smemAddr(&small.oFull));
                    }
                }
            } else if (!StateOnly && electOne()) {
                // whichever is ready: neither the scores of the next chunk nor the outputs of this one keep the other waiting
                Turn scoreTurn, outTurn;
                uint32_t idle = 0;
                for (int next = 0, u = 0; u < count && alive;) {
                    bool worked = false;
                    if (next < count && next <= u + 1 && testPhase(smemAddr(&small.fullK[scoreTurn.at]), scoreTurn.parity) && testPhase(smemAddr(&small.fullQ[scoreTurn.at]), scoreTurn.parity) &&
                        (next < 2 || testPhase(smemAddr(&small.pFree[next & 1]), ((next >> 1) - 1) & 1))) {
                        fenceAfter();
                        const uint32_t at = tiles + scoreTurn.at * kStageBytes;
                        const uint64_t q = swizzledDescriptor(at), k = swizzledDescriptor(at + kHalves * kTile);
#pragma unroll 2
                        for (int i = 0; i < 4 * kHalves; ++i) {
                            const uint64_t step = (i / 4) * (kTile >> 4) + (i % 4) * 2;
                            product(tmem + kP + (next & 1) * kC, q + step, k + step, kScores, i > 0);
                        }
                        commitTo(smemAddr(&small.pFull[next & 1]));
                        commitTo(smemAddr(&small.freeK[scoreTurn.at]));
                        commitTo(smemAddr(&small.freeQ[scoreTurn.at]));
                        ++next;
                        scoreTurn.step(kStages);
                        worked = true;
                    }
                    // V is clean behind the row's end, and has been read for its weighted form, once the state says so
                    if (u < next && testPhase(smemAddr(&small.pReady[u & 1]), (u >> 1) & 1) && testPhase(smemAddr(&small.vRead[outTurn.at]), outTurn.parity) &&
                        (u == 0 || testPhase(smemAddr(&small.oFree), (u - 1) & 1))) {
                        fenceAfter();
                        const uint64_t v = swizzledDescriptor(tiles + outTurn.at * kStageBytes + 2 * kHalves * kTile);
#pragma unroll 2
                        for (int i = 0; i < kC / 16; ++i) productTmem(tmem + kO2, tmem + kP + (u & 1) * kC + (i / 4) * 64 + (i % 4) * 8, v + i * 128, kOutputs, i > 0);
                        commitTo(smemAddr(&small.pFree[u & 1]));
                        commitTo(smemAddr(&small.oFull));
                        commitTo(smemAddr(&small.freeV[outTurn.at]));
                        ++u;
                        outTurn.step(kStages);
                        worked = true;
                    }
                    idle = worked ? 0 : idle + 1;
                    alive = idle < kSpinLimit;
                }
            }
            __syncwarp();
            // products go on after a wait that gave up, on whatever the operands hold; they end before the tensor memory is freed
            uint64_t &done = small.productsDone[warp - kStateProducts];
            if (electOne()) commitTo(smemAddr(&done));
            __syncwarp();
            waitSuspended(smemAddr(&done), 0);
            alive = __all_sync(0xffffffffu, alive);
        }
    } else if (warp < kFirstOutput) {
        giveRegisters<72>();
        if (!StateOnly) {
            // The thread's token, and the half of the columns that it takes: their scores lie in 64 columns of tensor memory, whose first 32 take what becomes of them.
            const int quarter = warp & 3, half = warp >> 2, i = 32 * quarter + lane;
            auto empty = [&](int block) { return reverse ? block < quarter : block > quarter; };
            for (int u = 0; u < count; ++u) {
                const int n = tokensOf(span.chunkAt(u, reverse));
                const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16) + kP + (u & 1) * kC + half * 64;
                // f(block, scores times the decays) for the two blocks of 32 columns that are not empty
                auto eachBlock = [&](auto f) {
#pragma unroll 1
                    for (int e = 0; e < 2; ++e) {
                        const int block = 2 * half + e;
                        if (empty(block)) continue;
                        uint32_t r[32];
                        loadTmem32(lanes + e * 32, r);
                        loadsDone();
                        if (block == quarter) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const int apart = reverse ? j - lane : lane - j;
                                r[j] = apart >= 0 ? __float_as_uint(__uint_as_float(r[j]) * small.scaledPowers[max(apart, 0)]) : 0u;
                            }
                        } else {
                            const float power = small.powers[reverse ? block * 32 - i : i - block * 32 - 31];
                            const Pair row = pairOf(power, power);
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                const float4 c = *reinterpret_cast<const float4 *>(&small.columnPowers[j]);
                                const float2 a = floatsOf(mul2(mul2(pairOf(r[j], r[j + 1]), pairOf(c.x, c.y)), row)), b2 = floatsOf(mul2(mul2(pairOf(r[j + 2], r[j + 3]), pairOf(c.z, c.w)), row));
                                r[j] = __float_as_uint(a.x);
                                r[j + 1] = __float_as_uint(a.y);
                                r[j + 2] = __float_as_uint(b2.x);
                                r[j + 3] = __float_as_uint(b2.y);
                            }
                        }
                        if (reverse && block * 32 + 32 > n) {   // tokens behind the row's end may hold anything
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (block * 32 + j >= n) r[j] = 0u;
                        }
                        f(e, r);
                    }
                };
                wait(small.pFull[u & 1], (u >> 1) & 1);
                fenceAfter();
                float up = 1.f;
                if constexpr (kHalf) {
                    float most = 0.f;
                    eachBlock([&](int, const uint32_t(&r)[32]) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) most = fmaxf(most, fabsf(__uint_as_float(r[j])));
                    });
                    const uint32_t own = exponentBits(most);
                    small.rowPeaks[u & 1][half][i] = static_cast<uint8_t>(own);
                    groupBarrier(kLanesMeet + quarter, 64);
                    up = toTopOfHalf(max(own, static_cast<uint32_t>(small.rowPeaks[u & 1][half ^ 1][i])));
                    if (half == 0) small.rowScale[u % 3][i] = static_cast<uint8_t>(exponentBits(up));
                }
                eachBlock([&](int e, const uint32_t(&r)[32]) {
                    uint32_t words[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) words[j] = kHalf ? pack2<T>(mul2(pairOf(r[2 * j], r[2 * j + 1]), pairOf(up, up))) : pack2<T>(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                    storeTmem16(lanes + e * 16, words);
                });
#pragma unroll 1
                for (int e = 0; e < 2; ++e)   // the scores of these are all read by now
                    if (empty(2 * half + e)) storeTmem16(lanes + e * 16, {});
                tmemStoresDone();
                fenceBefore();
                arriveWarp(small.pReady[u & 1]);
            }
        }
    } else if (warp < kFirstState) {
        giveRegisters<56>();
        if (!StateOnly) {
            const int quarter = warp & 3, i = 32 * quarter + lane;   // the thread's token
            const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
            for (int u = 0; u < count; ++u) {
                const uint32_t parity = u & 1;
                const int chunk = span.chunkAt(u, reverse), n = tokensOf(chunk);
                wait(small.oFull, parity);
                fenceAfter();
                const bool live = i < n, in = chunk * kC + i < p.tokens && alive && p.out, bad = __any_sync(0xffffffffu, small.lastBad > static_cast<uint32_t>(u));
                const float inter = live ? p.outScale * small.powers[reverse ? n - 1 - i : i + 1] * (kHalf ? small.stateScale[parity] : 1.f) : 0.f;
                float back = 1.f;
                if constexpr (kHalf) back = __uint_as_float((254u - small.rowScale[u % 3][i]) << 23);
                const size_t row = ((static_cast<size_t>(b) * p.tokens + chunk * kC + i) * p.heads + h) * p.value;
                // One round of code for all parts: warps of every role fetch instructions from the same cache, and unrolled they halve one another's speed.
#pragma unroll 1
                for (int part = 0; part < 4; ++part) {
                    uint32_t o1[16], o2[16];
                    loadTmem16(lanes + kO1 + part * 16, o1);
                    loadTmem16(lanes + kO2 + part * 16, o2);
                    loadsDone();
                    if (part == 3) {
                        fenceBefore();
                        if (!bad) arriveWarp(small.oFree);
                    }
                    const int col = slice * kCols + part * 16;
                    if (!in || col >= p.value) continue;
                    float out[16];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const Pair scaled = kHalf ? mul2(pairOf(o2[j], o2[j + 1]), pairOf(back, back)) : pairOf(o2[j], o2[j + 1]);
                        const float2 v = floatsOf(fma2(pairOf(o1[j], o1[j + 1]), pairOf(inter, inter), scaled));
                        out[j] = live ? v.x : 0.f;
                        out[j + 1] = live ? v.y : 0.f;
                    }
                    if (bad && live) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (small.badFrom[u % 3][part * 16 + j] >= badKey(u, i, reverse)) out[j] = __int_as_float(0x7fffffff);
                    }
                    auto sector = [](void *to, const uint32_t(&w)[8]) {   // a sector of memory a thread
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                     : "memory");
                    };
                    if constexpr (How == Stores::Packed) {
                        uint32_t w[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = pack2<T>(out[2 * j], out[2 * j + 1]);
                        sector(static_cast<T *>(p.out) + row + col, w);
                    } else if constexpr (How == Stores::Floats) {
#pragma unroll
                        for (int half = 0; half < 16; half += 8) {
                            uint32_t w[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(out[half + j]);
                            if (col + half < p.value) sector(static_cast<float *>(p.out) + row + col + half, w);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            if (col + j >= p.value) continue;
                            if (p.outFloat) static_cast<float *>(p.out)[row + col + j] = out[j];
                            else static_cast<T *>(p.out)[row + col + j] = fromFloat<T>(out[j]);
                        }
                    }
                }
                // The state writes of chunk u + 3 what it writes of chunk u, once the outputs of chunk u have let go of their products.
                if (bad) arriveWarp(small.oFree);
            }
        }
    } else {
        takeRegisters<120>();
        // The thread's row of the state and its columns of it: a half with 128 keys; a quarter with 64, whose rows stand twice in KV, so that all eight warps
        // have work (8 x 4096 tokens, 16 heads of 64: 66.4 -> 63.6 us against halves for four of the warps).
        constexpr int kMine = DK == 64 ? 16 : 32;
        const int quarter = warp & 3, d = (32 * quarter + lane) % DK, mine = ((warp - kFirstState) >> 2) * (128 / DK) + 32 * quarter / DK;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
        const int stid = tid - 32 * kFirstState;
        const size_t head = static_cast<size_t>(b) * p.heads + h, stateSize = static_cast<size_t>(p.key) * p.value;
        const int col = slice * kCols + mine * kMine;
        Pair s[kMine / 2];
        const float *in = segments.count > 1 ? (StateOnly ? nullptr : segments.states + (head * segments.count + segment) * stateSize) : p.stateIn ? p.stateIn + head * stateSize : nullptr;
        const int inRow = segments.count > 1 ? p.value : p.stateRow, inCol = segments.count > 1 ? 1 : p.stateCol;
        const float inScale = segments.count > 1 ? 1.f : p.inScale;
#pragma unroll
        for (int j = 0; j < kMine / 2; ++j) s[j] = pairOf(0.f, 0.f);
        if (in && d < p.key) {
            const float *from = in + static_cast<size_t>(d) * inRow + static_cast<size_t>(col) * inCol;
            if (inCol == 1 && p.value % 4 == 0 && (reinterpret_cast<uintptr_t>(in) & 15) == 0) {
#pragma unroll
                for (int j = 0; j < kMine / 2; j += 2) {
                    if (col + 2 * j >= p.value) continue;
                    const float4 v = *reinterpret_cast<const float4 *>(from + 2 * j);
                    s[j] = pairOf(v.x * inScale, v.y * inScale);
                    s[j + 1] = pairOf(v.z * inScale, v.w * inScale);
                }
            } else
#pragma unroll
            for (int j = 0; j < kMine / 2; ++j, from += 2 * inCol)
                s[j] = pairOf(col + 2 * j < p.value ? inScale * from[0] : 0.f, col + 2 * j + 1 < p.value ? inScale * from[inCol] : 0.f);
        }

        auto publish = [&](int u) {   // the state in front of chunk u, as the B operand of O1
            float up = 1.f;
            if constexpr (kHalf) {
                float most = 0.f;
#pragma unroll
                for (int j = 0; j < kMine / 2; ++j) {
                    const float2 v = floatsOf(s[j]);
                    most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
                const uint32_t peak = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
                if (lane == 0) small.statePeaks[u & 1][stid >> 5] = __uint_as_float(peak);
                groupBarrier(kStateMeets, 32 * kStateWarps);
                most = 0.f;
#pragma unroll
                for (int w = 0; w < kStateWarps; ++w) most = fmaxf(most, small.statePeaks[u & 1][w]);
                up = toTopOfHalf(exponentBits(most));
                if (stid == 0) small.stateScale[u & 1] = 1.f / up;
            }
#pragma unroll
            for (int c = 0; c < kMine / 8; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = kHalf ? pack2<T>(mul2(s[4 * c + j], pairOf(up, up))) : pack2<T>(s[4 * c + j]);
                storeShared(sTile + d * 128 + (((mine * (kMine / 8) + c) ^ (d & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
            fenceAsyncProxy();
            arriveWarp(small.sReady);
        };

        float down = 1.f, downNext = 1.f;   // one over the scales of the weighted V of half, of this chunk and the next
        auto advance = [&](int u) {   // the state behind chunk u
            const float keep = small.powers[tokensOf(span.chunkAt(u, reverse))];
#pragma unroll
            for (int part = 0; part < kMine / 16; ++part) {
                uint32_t r[16], low[16];
                const uint32_t from = lanes + kKV + mine * kMine + part * 16;
                loadTmem16(from, r);
                loadTmem16(from + kCols, low);
                loadsDone();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const Pair high = pairOf(r[2 * j], r[2 * j + 1]), rest = pairOf(low[2 * j], low[2 * j + 1]);
                    // the power of two that V was scaled by taken out again, exactly
                    s[part * 8 + j] = fma2(s[part * 8 + j], pairOf(keep, keep), kHalf ? fma2(rest, pairOf(down / 2048, down / 2048), mul2(high, pairOf(down, down))) : add2(high, rest));
                }
            }
            fenceBefore();
        };
        const int token = stid >> 1;   // of whose 64 values this thread weights 32
        const uint32_t place = token * 128, piece = (stid & 1) * 4;
        auto pieceAt = [&](int c) { return place + (((piece + c) ^ (token & 7)) << 4); };
        auto weightOf = [&](int n) { return token < n ? small.powers[reverse ? token + 1 : n - 1 - token] : 0.f; };
        auto less = [&](Pair x, uint32_t term) {   // what a term leaves; exact
            const float2 t = unpack2<T>(term);
            return fma2(pairOf(t.x, t.y), pairOf(-1.f, -1.f), x);
        };
        uint32_t hi[4][4], mid[4][4], low[Third ? 4 : 1][4];   // the terms of the next chunk's weighted V
        Turn turn;
        auto weigh = [&](int u) {
            const uint32_t at = tiles + turn.at * kStageBytes;
            const int chunk = span.chunkAt(u, reverse), n = tokensOf(chunk);
            wait(small.fullV[turn.at], turn.parity);
            if (n < kC && chunk * kC + n < p.tokens) {   // K and V behind the row's end may hold anything, and zero times that is not zero
                wait(small.fullK[turn.at], turn.parity);
                for (int i = (kHalves * kC + n) * 8 + stid; i < (2 * kHalves + 1) * kC * 8; i += 32 * kStateWarps)
                    if ((i / 8) % kC >= n) storeShared(at + i * 16, 0u, 0u, 0u, 0u);
                fenceAsyncProxy();
                groupBarrier(kStateMeets, 32 * kStateWarps);
            }
            float w = weightOf(n);
#pragma unroll
            for (int c = 0; c < 4; ++c) loadShared(at + 2 * kHalves * kTile + pieceAt(c), hi[c]);
            if constexpr (kHalf) {   // to the top of half's range
                __half2 most = __float2half2_rn(0.f);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) most = __hmax2(most, __habs2(*reinterpret_cast<const __half2 *>(&hi[c][j])));
                const uint32_t own = __reduce_max_sync(0xffffffffu, __float_as_uint(w * fmaxf(__low2float(most), __high2float(most))));
                if (lane == 0) small.valuePeaks[u & 1][stid >> 5] = __uint_as_float(own);
                groupBarrier(kStateMeets, 32 * kStateWarps);
                float peak = 0.f;
#pragma unroll
                for (int i = 0; i < kStateWarps; ++i) peak = fmaxf(peak, small.valuePeaks[u & 1][i]);
                const float up = toTopOfHalf(exponentBits(peak));
                downNext = 1.f / up;
                w *= up;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 x = unpack2<T>(hi[c][j]);
                    const Pair weighted = mul2(pairOf(x.x, x.y), pairOf(w, w));
                    hi[c][j] = pack2<T>(weighted);
                    Pair rest = less(weighted, hi[c][j]);
                    if constexpr (kHalf) rest = mul2(rest, pairOf(2048.f, 2048.f));
                    mid[c][j] = pack2<T>(rest);
                    if constexpr (Third) low[c][j] = pack2<T>(less(rest, mid[c][j]));
                }
        };
        if (count > 0) weigh(0);
        for (int u = 0; u < count; ++u) {
            const uint32_t parity = u & 1;
            if (u > 0) advance(u - 1);
            down = downNext;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                storeShared(weightedV + pieceAt(c), hi[c][0], hi[c][1], hi[c][2], hi[c][3]);
                storeShared(weightedV + kTile + pieceAt(c), mid[c][0], mid[c][1], mid[c][2], mid[c][3]);
                if constexpr (Third) storeShared(weightedV + 2 * kTile + pieceAt(c), low[c][0], low[c][1], low[c][2], low[c][3]);
            }
            fenceAsyncProxy();
            arriveWarp(small.vReady);
            // under the product of this chunk: the state in front of it, and the terms of the next one
            if (!StateOnly) {
                if (u > 0) wait(small.sFree, parity ^ 1u);
                publish(u);
            }
            if (!StateOnly) {
                // A vote: with a branch a thread 8 x 4096 tokens of 16 heads of 64 take 68 us, so 64.  Behind the state's publication: in front of it, 128 elements a head take 163 for 161.
                uint32_t sums[4] = {};
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) addZeroTimes<T>(sums[j], mid[c][j]);
                if (__any_sync(0xffffffffu, ((sums[0] | sums[1] | sums[2] | sums[3]) & 0x7fff7fffu) != 0u)) {
                    clean<T>(tiles + turn.at * kStageBytes + 2 * kHalves * kTile + place, token & 7, piece, small.badFrom[u % 3], badKey(u, token, reverse));
                    small.lastBad = u + 1;
                    fenceAsyncProxy();
                }
                arriveWarp(small.vRead[turn.at]);
            }

            turn.step(kStages);
            if (u + 1 < count) weigh(u + 1);
            wait(small.kvFull, parity);
            fenceAfter();
        }
        if (count > 0) advance(count - 1);
        float *last = StateOnly ? segments.states + (head * segments.count + segment) * stateSize : segments.count > 1 || !p.stateOut ? nullptr : p.stateOut + head * stateSize;
        if (last && alive) {
            const int outRow = StateOnly ? p.value : p.stateRow, outCol = StateOnly ? 1 : p.stateCol;
            const float scale = StateOnly ? 1.f : p.finalScale;
            float *to = last + static_cast<size_t>(d) * outRow + static_cast<size_t>(col) * outCol;
            if (d < p.key) {
                if (outCol == 1 && p.value % 4 == 0 && (reinterpret_cast<uintptr_t>(last) & 15) == 0) {
#pragma unroll
                    for (int j = 0; j < kMine / 2; j += 2)
                        if (col + 2 * j < p.value)
                            *reinterpret_cast<float4 *>(to + 2 * j) = make_float4(floatsOf(s[j]).x * scale, floatsOf(s[j]).y * scale, floatsOf(s[j + 1]).x * scale, floatsOf(s[j + 1]).y * scale);
                } else {
#pragma unroll
                    for (int j = 0; j < kMine; ++j)
                        if (col + j < p.value) to[static_cast<size_t>(j) * outCol] = (j & 1 ? floatsOf(s[j / 2]).y : floatsOf(s[j / 2]).x) * scale;
                }
            }
        }
    }
    if (!alive && lane == 0) small.failed = 1;
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
    if (warp == kStateProducts) freeTmem<1>(tmem, 512);
    if (tid == 0 && small.failed) atomicExch(status, 1);
}

// From the ends of the segments on their own to their beginnings: one thread for each element of a state, segment after segment, eight of them in flight.  The powers of the decay
// are made once a CTA: in 64 bits and by every thread, they took 35 us for 16 segments (1 x 16384 tokens of 8 heads of 64) in place of 6.
__global__ void __launch_bounds__(256) joinSegments(const __grid_constant__ Pass p, const Segments segments) {
    constexpr int kAtOnce = 8;
    __shared__ float powers[kMaxSegments];   // of the decay over a segment's tokens; below zero for one without any
    const int h = blockIdx.y, b = blockIdx.z, size = p.key * p.value, e = blockIdx.x * 256 + threadIdx.x;
    waitForPredecessor();
    letDependentsStart();
    const int length = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
    for (int i = threadIdx.x; i < segments.count; i += 256) {
        const int tokens = Span(length, i, segments.chunks).tokens(length, p.reverse);
        powers[i] = tokens > 0 ? static_cast<float>(exp(tokens * static_cast<double>(p.logDecay[h]))) : -1.f;
    }
    __syncthreads();
    if (e >= size) return;
    const size_t head = static_cast<size_t>(b) * p.heads + h, at = head * size + static_cast<size_t>(e / p.value) * p.stateRow + static_cast<size_t>(e % p.value) * p.stateCol;
    float state = p.stateIn ? p.inScale * p.stateIn[at] : 0.f;
    float *own = segments.states + head * segments.count * size + e;
    for (int first = 0; first < segments.count; first += kAtOnce) {
        float added[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (first + i < segments.count && powers[first + i] >= 0.f) added[i] = own[static_cast<size_t>(first + i) * size];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (first + i >= segments.count) break;
            own[static_cast<size_t>(first + i) * size] = state;
            if (powers[first + i] >= 0.f) state = fmaf(state, powers[first + i], added[i]);
        }
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

// From 16 tokens on where all CTAs find an SM, else from 32 on: a launch takes 8 to 14 us a round whatever the number of tokens up to 128, token by token a token takes 0.45 to 0.6 us with few
// heads (8 of 64: 16 tokens 10.8 for 8.6) and less than its share with many (1024 of 128: 31 tokens 123 us, one chunk 171).
// Segments by these estimates, in microseconds, of measured launches: a launch begins and ends in 8, a chunk takes 2.2, 1.3 where only the state is wanted, joining 4.  Eight chunks of 48
// heads: 26 in one, 31 in three segments; 128 chunks of 8 heads: 290 in one, 48 in sixteen.
ChunkPlan planChunks(const Pass &p, int type) {
    ChunkPlan plan{false, 1, (p.tokens + kC - 1) / kC};
    const int chunks = plan.segmentChunks, sms = currentDevice().sms;
    const int64_t ctas = std::max<int64_t>(1, static_cast<int64_t>((p.value + kCols - 1) / kCols) * p.heads * p.batch);
    plan.taken = type != RXMET_TYPE_F32 && p.tokens >= (ctas <= sms ? 16 : 32) && encodeTiled() != nullptr;
    if (!plan.taken) return plan;
    const auto rounds = [&](int segments) { return static_cast<double>((ctas * segments + sms - 1) / sms); };
    double best = rounds(1) * (8 + 2.2 * chunks);
    for (int segments = 2; segments <= chunks / 2 && segments <= kMaxSegments && ctas * segments <= 2 * sms; ++segments) {
        const int each = (chunks + segments - 1) / segments;
        const double time = rounds(segments) * (16 + 3.5 * each) + 4;
        if (time >= best) continue;
        best = time;
        plan.segmentChunks = each;
        plan.segments = (chunks + each - 1) / each;
    }
    return plan;
}

bool chunksCanCopy(const Pass &p) { return copies(p.q, p.batch, p.tokens) && copies(p.k, p.batch, p.tokens) && copies(p.v, p.batch, p.tokens); }

void launchChunks(const Pass &p, int type, const ChunkPlan &plan, float *states, cudaStream_t st) {
    const bool bf16 = type == RXMET_TYPE_BF16;
    bool ok = true;
    bindContext();
    const CUtensorMap q = tokenMap(p.q, p.batch, p.tokens, p.key, bf16, ok), k = tokenMap(p.k, p.batch, p.tokens, p.key, bf16, ok), v = tokenMap(p.v, p.batch, p.tokens, p.value, bf16, ok);
    const bool wide = p.value % (p.outFloat ? 8 : 16) == 0 && alignedTo(p.out, 32);   // parts of a row start on 32 bytes
    if (!ok) fail(RXMET_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    const Segments segments{plan.segments, plan.segmentChunks, states};
    const dim3 grid((p.value + kCols - 1) / kCols * plan.segments, p.heads, p.batch);
    auto run = [&](auto kernel, const char *name) {
        ensureDynamicSmem(reinterpret_cast<const void *>(kernel), kShared);
        {
            KernelTimer timer__(name, st);
            launchDependent(kernel, grid, kThreads, kShared, st, p, q, k, v, segments, waitStatus());
        }
        afterLaunch(name);
    };
    auto both = [&](auto t, auto dk) {
        using T = decltype(t);
        constexpr int DK = decltype(dk)::value;
        constexpr bool kThree = std::is_same<T, __nv_bfloat16>::value;
        auto outputs = [&](auto third) {
            constexpr bool Third = decltype(third)::value;
            run(!wide        ? decayedChunks<T, DK, Third, false, Stores::Elements>
                : p.outFloat ? decayedChunks<T, DK, Third, false, Stores::Floats>
                             : decayedChunks<T, DK, Third, false, Stores::Packed>,
                "decayedChunks");
        };
        // Three bfloat16 terms of the weighted V where the state is an output; two, 2^-17, where it only feeds products that round it to 2^-9.
        if (plan.segments > 1) {
            run(p.stateOut ? decayedChunks<T, DK, kThree, true, Stores::Elements> : decayedChunks<T, DK, false, true, Stores::Elements>, "decayedChunksState");
            {
                KernelTimer timer__("joinSegments", st);
                launchDependent(joinSegments, dim3((p.key * p.value + 255) / 256, p.heads, p.batch), 256, 0, st, p, segments);
            }
            afterLaunch("joinSegments");
            if (p.out) outputs(std::false_type{});
        } else if (p.stateOut) outputs(std::integral_constant<bool, kThree>{});
        else outputs(std::false_type{});
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
