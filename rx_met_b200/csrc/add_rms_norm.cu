// Residual addition with a root-mean-square norm (to the input's type, or to 8-bit codes with a scale for each row), and its gradient.
//
// One pass over the data: a team of 8 to 512 threads holds a row in registers, so that the sum, the largest magnitude and the output need no
// second read.  A team walks over rows, which keeps the weights in registers.  The rows come through a ring in shared memory that bulk copies fill two to four rounds
// ahead.  With loads to registers one row ahead in its place, 8192 x 4096 bfloat16 take 66 us for 60 (forward with codes) and 105 for 78 (gradients), at the same 16 elements a thread.
// Sums run in 32 bits: a thread's own elements in order, lanes as a tree, warps in order, so that results do not depend on the grid.
//
// Bound: HBM for codes (8192 x 4096 bfloat16 43 us, 5.5 TB/s) and the forward (49.5 us, 5.4 TB/s); issue and the barrier of a team's sum for the gradients (78 us, 4.3 TB/s).
#include <algorithm>

#include "common.h"
#include "dependent_launch.cuh"
#include "cluster_device.cuh"
#include "element_types.cuh"
#include "umma_device.cuh"

namespace rxmet {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kMaxCoded = 131071;   // of rows that are only coded: as many as a product of codes takes
constexpr int kMaxThreads = 512, kMaxWarps = kMaxThreads / 32;

// The rows of a round (one for each team of a CTA) of up to four arrays, in shared memory.  Bulk copies start and end on 16 bytes, so a copy takes the few bytes
// around what it wants as well; they share a 16-byte unit, and so a page, with bytes that it does want.
struct Ring {
    static constexpr int kMaxDepth = 4;
    int depth = 0;             // 0: no ring
    uint32_t arrayBytes = 0;   // of one array in one stage
};
struct Source {
    const void *data;
    int64_t pitch;   // elements
};

struct NormRows {
    int64_t rows;
    int width, team;   // team: its threads, a power of two up to 32 or a multiple of it
    Ring ring;
    const void *x, *residual, *weight;
    int64_t xPitch, residualPitch;
    int weightType;
    float eps;
    void *total, *y;
    float *rms;
    int8_t *codes;
    int64_t codesPitch;
    float *scale;
};

__device__ __forceinline__ float larger(float a, float b) {   // a NaN wins
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The place of a thread in its team.  Teams of a CTA work on rows of their own; those of several warps meet at a barrier of their own, after which every warp adds up
// what the others have left, a lane for each.
struct Team {
    int size, index, count, rank;
    __device__ __forceinline__ explicit Team(int threads) : size(threads), index(threadIdx.x / threads), count(blockDim.x / threads), rank(threadIdx.x - index * threads) {}
    // `slot` alternates between two arrays from row to row, so that one barrier is enough.
    template <class F>
    __device__ __forceinline__ float reduce(float v, float (*shared)[kMaxWarps], int slot, F f) const {
        if (size < 32) {
            for (int d = size / 2; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
            return v;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
        if (size == 32) return v;
        const int lane = threadIdx.x & 31;
        if (lane == 0) shared[slot][threadIdx.x >> 5] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(size) : "memory");
        v = (lane & (kMaxWarps - 1)) < size / 32 ? shared[slot][index * size / 32 + (lane & (kMaxWarps - 1))] : 0.f;
#pragma unroll
        for (int d = kMaxWarps / 2; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    }
    __device__ __forceinline__ float sum(float v, float (*shared)[kMaxWarps], int slot) const {
        return reduce(v, shared, slot, [](float a, float b) { return a + b; });
    }
    __device__ __forceinline__ float most(float v, float (*shared)[kMaxWarps], int slot) const {
        return reduce(v, shared, slot, [](float a, float b) { return larger(a, b); });
    }
};

__device__ __forceinline__ float weightAt(const void *weight, int type, int i) {
    if (type == RXMET_TYPE_F32) return static_cast<const float *>(weight)[i];
    if (type == RXMET_TYPE_BF16) return toFloat(static_cast<const __nv_bfloat16 *>(weight)[i]);
    return toFloat(static_cast<const __half *>(weight)[i]);
}

// W neighbouring elements in 32 bits, two to a register pair: one operation for both.
template <int W>
struct Lanes {
    Pair v[W / 2];
    template <class F>
    __device__ __forceinline__ static Lanes of(F f) {
        Lanes r;
#pragma unroll
        for (int i = 0; i < W / 2; ++i) r.v[i] = f(i);
        return r;
    }
    __device__ __forceinline__ Lanes operator+(const Lanes &o) const { return of([&](int i) { return add2(v[i], o.v[i]); }); }
    __device__ __forceinline__ Lanes operator*(const Lanes &o) const { return of([&](int i) { return mul2(v[i], o.v[i]); }); }
    __device__ __forceinline__ Lanes operator*(float f) const { return of([&](int i) { return mul2(v[i], pairOf(f, f)); }); }
    __device__ __forceinline__ Lanes plus(const Lanes &a, const Lanes &b) const { return of([&](int i) { return fma2(a.v[i], b.v[i], v[i]); }); }
    __device__ __forceinline__ Lanes plus(const Lanes &a, float f) const { return of([&](int i) { return fma2(a.v[i], pairOf(f, f), v[i]); }); }
    __device__ __forceinline__ float total() const {
        Pair sum = v[0];
#pragma unroll
        for (int i = 1; i < W / 2; ++i) sum = add2(sum, v[i]);
        return floatsOf(sum).x + floatsOf(sum).y;
    }
    __device__ __forceinline__ float at(int j) const { return j & 1 ? floatsOf(v[j / 2]).y : floatsOf(v[j / 2]).x; }
    __device__ __forceinline__ void set(int j, float f) { v[j / 2] = j & 1 ? pairOf(floatsOf(v[j / 2]).x, f) : pairOf(f, floatsOf(v[j / 2]).y); }
};
template <>
struct Lanes<1> {
    float v;
    __device__ __forceinline__ Lanes operator+(const Lanes &o) const { return {v + o.v}; }
    __device__ __forceinline__ Lanes operator*(const Lanes &o) const { return {v * o.v}; }
    __device__ __forceinline__ Lanes operator*(float f) const { return {v * f}; }
    __device__ __forceinline__ Lanes plus(const Lanes &a, const Lanes &b) const { return {fmaf(a.v, b.v, v)}; }
    __device__ __forceinline__ Lanes plus(const Lanes &a, float f) const { return {fmaf(a.v, f, v)}; }
    __device__ __forceinline__ float total() const { return v; }
    __device__ __forceinline__ float at(int) const { return v; }
    __device__ __forceinline__ void set(int, float f) { v = f; }
};
template <int W>
__device__ __forceinline__ Lanes<W> allOf(float f) {
    Lanes<W> r;
    if constexpr (W == 1) r.v = f;
    else r = Lanes<W>::of([&](int) { return pairOf(f, f); });
    return r;
}
template <class T, int W>
__device__ __forceinline__ Lanes<W> loadLanes(const T *from) {
    const Pack<T, W> in = *reinterpret_cast<const Pack<T, W> *>(from);
    Lanes<W> r;
    if constexpr (W == 1) {
        r.v = toFloat(in.v[0]);
    } else if constexpr (sizeof(T) == 4) {
        r = Lanes<W>::of([&](int i) { return pairOf(in.v[2 * i], in.v[2 * i + 1]); });
    } else {
        const uint32_t *words = reinterpret_cast<const uint32_t *>(&in);
        r = Lanes<W>::of([&](int i) {
            const float2 v = unpack2<T>(words[i]);
            return pairOf(v.x, v.y);
        });
    }
    return r;
}
template <class T, int W>
__device__ __forceinline__ void storeLanes(T *to, const Lanes<W> &l) {
    Pack<T, W> out;
    if constexpr (W == 1) {
        out.v[0] = fromFloat<T>(l.v);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < W; ++j) out.v[j] = l.at(j);
    } else {
        uint32_t *words = reinterpret_cast<uint32_t *>(&out);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) words[i] = pack2<T>(l.v[i]);
    }
    *reinterpret_cast<Pack<T, W> *>(to) = out;
}

// One CTA's side of a ring.
template <class T, int ARRAYS>
struct RingReader {
    const Source *sources;
    const Ring ring;
    int64_t rows;
    int width, teams;
    uint64_t *full, *freed;
    uint8_t *base;
    umma::Turn turn;       // the stage that is read
    umma::Turn ahead;      // the stage that is asked for next
    __device__ __forceinline__ uint32_t stageBytes() const { return ring.arrayBytes * ARRAYS; }
    // Whether the rows of a round lie one behind the other in memory, and so come as one copy.
    __device__ __forceinline__ bool together(int a) const { return sources[a].pitch == width; }
    __device__ __forceinline__ uint32_t slot() const { return (static_cast<uint32_t>(width * sizeof(T)) + 15) / 16 * 16 + 16; }   // of a row on its own
    // Asks for the rows from row0 on; all lanes of one warp.
    __device__ __forceinline__ void ask(int64_t row0) {
        const int lane = threadIdx.x & 31, here = static_cast<int>(min(static_cast<int64_t>(teams), rows - row0));
        if (ahead.again) umma::waitSuspended(umma::smemAddr(&freed[ahead.at]), ahead.parity ^ 1u);
        const uint32_t bar = umma::smemAddr(&full[ahead.at]), to = umma::smemAddr(base) + ahead.at * stageBytes();
        auto each = [&](auto f) {
#pragma unroll
            for (int a = 0; a < ARRAYS; ++a) {
                if (!sources[a].data) continue;
                const int copies = together(a) ? 1 : here, rowsOf = together(a) ? here : 1;
                for (int i = lane; i < copies; i += 32) {
                    const uintptr_t from = reinterpret_cast<uintptr_t>(static_cast<const T *>(sources[a].data) + (row0 + i) * sources[a].pitch);
                    const uintptr_t begin = from & ~static_cast<uintptr_t>(15), end = (from + static_cast<uintptr_t>(rowsOf) * width * sizeof(T) + 15) & ~static_cast<uintptr_t>(15);
                    f(to + a * ring.arrayBytes + i * slot(), begin, static_cast<uint32_t>(end - begin));
                }
            }
        };
        uint32_t bytes = 0;
        each([&](uint32_t, uintptr_t, uint32_t n) { bytes += n; });
        bytes = __reduce_add_sync(0xffffffffu, bytes);
        if (lane == 0) cluster::arriveExpect(bar, bytes);
        __syncwarp();
        each([&](uint32_t at, uintptr_t begin, uint32_t n) {
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(at), "l"(begin), "r"(n), "r"(bar) : "memory");
        });
        ahead.step(ring.depth);
    }
    // A team's row of array a in the stage that is read.  Aligned: all rows start on 16 bytes.
    template <bool Aligned>
    __device__ __forceinline__ const T *row(int a, int64_t row0, int team) const {
        const bool joint = together(a);
        uint32_t at = turn.at * stageBytes() + a * ring.arrayBytes + team * (joint ? width * static_cast<uint32_t>(sizeof(T)) : slot());
        // where in its 16 bytes the copy's first row starts: the low bits of its address
        if constexpr (!Aligned)
            at += (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(sources[a].data)) +
                   (static_cast<uint32_t>(row0) + (joint ? 0 : team)) * static_cast<uint32_t>(sources[a].pitch) * static_cast<uint32_t>(sizeof(T))) & 15u;
        return reinterpret_cast<const T *>(base + at);
    }
    __device__ __forceinline__ bool wait() const { return umma::waitSuspended(umma::smemAddr(&full[turn.at]), turn.parity); }
    __device__ __forceinline__ void done() {   // by every warp, once it has read its rows
        __syncwarp();
        if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(umma::smemAddr(&freed[turn.at])) : "memory");
        turn.step(ring.depth);
    }
};
// Barriers of a ring, and the bytes behind them.
struct RingSpace {
    uint64_t full[Ring::kMaxDepth], freed[Ring::kMaxDepth];
    __device__ __forceinline__ void init(int depth) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < depth; ++i) {
                cluster::initBarrier(&full[i], 1);
                cluster::initBarrier(&freed[i], blockDim.x / 32);
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
};

// Codes of a row whose 127 / peak is infinite, in place of those that a thread has just written: values and step are brought up by a power of two.  A step below the normal numbers may have
// been rounded down by so much that the largest values lie more than 127 of it from zero, or to zero itself.  The row is read again: such rows are rare, and with this in the kernel's
// registers 8192 x 4096 bfloat16 took 46.5 us for 44.
template <class T, int W>
__device__ __noinline__ void tinyCodes(const NormRows &p, int64_t row, float rms, float step, int first, int stride) {
    constexpr float kUp = 0x1p64f;
    const float inverse = step > 0.f ? 1.f / (step * kUp) : 0.f;
    for (int group = first; group < p.width; group += stride)
        for (int i = group; i < group + W; ++i) {
            float t = toFloat(static_cast<const T *>(p.x)[row * p.xPitch + i]);
            if (p.residual) t += toFloat(static_cast<const T *>(p.residual)[row * p.residualPitch + i]);
            t = t * rms * (p.weight ? weightAt(p.weight, p.weightType, i) : 1.f);
            p.codes[row * p.codesPitch + i] = static_cast<int8_t>(__float2int_rn(fminf(fmaxf(t * kUp * inverse, -127.f), 127.f)));
        }
}

// Codes of values over a step, whose inverse is given.  1.5 * 2^23 added, the low byte of the sum is the nearest integer, ties to even.  The quotient of the largest magnitude rounds to 127, so
// none lies beyond.
template <int W>
__device__ __forceinline__ Pack<int8_t, W> codesOf(const Lanes<W> &t, float inverse) {
    const Lanes<W> shifted = allOf<W>(12582912.f).plus(t, inverse);
    Pack<int8_t, W> out;
    if constexpr (W == 1) {
        out.v[0] = static_cast<int8_t>(__float_as_uint(shifted.v) & 0xffu);
    } else {
        uint32_t *words = reinterpret_cast<uint32_t *>(&out);
#pragma unroll
        for (int j = 0; j < W; j += 4)
            words[j / 4] = __byte_perm(__byte_perm(__float_as_uint(shifted.at(j)), __float_as_uint(shifted.at(j + 1)), 0x0040),
                                       __byte_perm(__float_as_uint(shifted.at(j + 2)), __float_as_uint(shifted.at(j + 3)), 0x0040), 0x5410);
    }
    return out;
}

// Ringed: rows come through the ring.  Else straight from memory: few rows, which have no next ones to fetch, and those too wide for a ring.
template <class T, int W, int ITEMS, bool Codes, bool Ringed>
__global__ void __launch_bounds__(kMaxThreads) __maxnreg__(W * ITEMS <= 8 ? 64 : W * ITEMS <= 16 ? (W > 1 ? 80 : 96) : 128) addRmsNorm(const __grid_constant__ NormRows p, int *status) {
    using Elements = Lanes<W>;
    __shared__ RingSpace space;
    extern __shared__ __align__(16) uint8_t stages[];
    __shared__ float sums[2][kMaxWarps], peaks[2][kMaxWarps];
    const Team team(p.team);
    const int first = team.rank * W, stride = team.size * W, width = p.width;
    const float perElement = 1.f / static_cast<float>(width);
    const bool norm = p.weight != nullptr;
    if constexpr (Ringed) space.init(p.ring.depth);
    waitForPredecessor();
    const int64_t step = static_cast<int64_t>(gridDim.x) * team.count, row0 = static_cast<int64_t>(blockIdx.x) * team.count;
    const Source sources[2] = {{p.x, p.xPitch}, {p.residual, p.residualPitch}};
    RingReader<T, 2> ring{sources, p.ring, p.rows, width, team.count, space.full, space.freed, stages};
    // all teams of a CTA go through the same number of rounds, because they shuffle together
    const int64_t rounds = row0 < p.rows ? (p.rows - row0 + step - 1) / step : 0;
    auto asks = [&](int64_t round) {   // the copies of a round, by the first warp
        if (threadIdx.x < 32 && round < rounds) ring.ask(row0 + round * step);
    };
    if constexpr (Ringed)
        for (int i = 0; i < p.ring.depth; ++i) asks(i);
    auto weightOf = [&](int i) {
        Elements w = allOf<W>(1.f);
        if (norm && first + i * stride < width)
#pragma unroll
            for (int j = 0; j < W; ++j) w.set(j, weightAt(p.weight, p.weightType, first + i * stride + j));
        return w;
    };
    Elements kept[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) kept[i] = weightOf(i);
    letDependentsStart();
    bool alive = true;
    for (int64_t round = 0; round < rounds; ++round) {
        const int slot = round & 1;
        const int64_t first0 = row0 + round * step, row = first0 + team.index;
        const bool real = row < p.rows;
        const T *x = static_cast<const T *>(p.x) + row * p.xPitch, *r = static_cast<const T *>(p.residual) + row * p.residualPitch;
        if constexpr (Ringed) {
            if (alive) alive = ring.wait();
            if (round > 0) asks(round - 1 + p.ring.depth);   // into the stage of the round before, which all warps have read or are about to
            x = ring.template row<(W > 1)>(0, first0, team.index);
            r = ring.template row<(W > 1)>(1, first0, team.index);
        }
        const int here = real ? width : 0;   // a row past the end is one of zeros
        Elements t[ITEMS], squares = allOf<W>(0.f);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            t[i] = allOf<W>(0.f);
            if (first + i * stride < here) {
                t[i] = loadLanes<T, W>(x + first + i * stride);
                if (p.residual) t[i] = t[i] + loadLanes<T, W>(r + first + i * stride);
            }
            squares = squares.plus(t[i], t[i]);
        }
        if constexpr (Ringed) ring.done();
        if (p.residual) {
            T *total = static_cast<T *>(p.total) + row * width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (first + i * stride < here) storeLanes<T, W>(total + first + i * stride, t[i]);
        }
        float rms = 1.f;
        if (norm) {
            rms = rsqrtf(fmaf(team.sum(squares.total(), sums, slot), perElement, p.eps));
            if (p.rms && first == 0 && real) p.rms[row] = rms;
        }
        float peak = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            t[i] = t[i] * rms * kept[i];   // zero beyond the row
            if constexpr (Codes)
#pragma unroll
                for (int j = 0; j < W; ++j) peak = larger(peak, fabsf(t[i].at(j)));
        }
        if constexpr (Codes) {
            const float most = team.most(peak, peaks, slot);
            const float inverse = most > 0.f ? 127.f / most : 0.f;
            if (real && first == 0) p.scale[row] = most / 127.f;
            int8_t *codes = p.codes + row * p.codesPitch;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const Pack<int8_t, W> out = codesOf(t[i], inverse);
                if (first + i * stride < here) *reinterpret_cast<Pack<int8_t, W> *>(codes + first + i * stride) = out;
            }
            if (isinf(inverse) && real) tinyCodes<T, W>(p, row, rms, most / 127.f, first, stride);
        } else {
            T *y = static_cast<T *>(p.y) + row * width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (first + i * stride < here) storeLanes<T, W>(y + first + i * stride, t[i]);
        }
    }
    if (!alive && (threadIdx.x & 31) == 0) atomicExch(status, 1);
}

// Codes of rows that a team's registers do not hold, without a norm: a CTA reads a row twice, the second time from L2, for its largest magnitude and for the codes.  Bound: the two readings
// (8192 x 28672 bfloat16 224 us, 3.1 TB/s of what a single reading and the codes would move).
constexpr int kWideThreads = 1024;
template <class T, int W>
__global__ void __launch_bounds__(kWideThreads) codeWideRows(const __grid_constant__ NormRows p) {
    __shared__ float peaks[2][kWideThreads / 32];
    const int first = threadIdx.x * W, stride = kWideThreads * W, lane = threadIdx.x & 31;
    waitForPredecessor();
    letDependentsStart();
    int slot = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, slot ^= 1) {
        const T *x = static_cast<const T *>(p.x) + row * p.xPitch, *r = static_cast<const T *>(p.residual) + row * p.residualPitch;
        auto sum = [&](int i) {
            const Lanes<W> t = loadLanes<T, W>(x + i);
            return p.residual ? t + loadLanes<T, W>(r + i) : t;
        };
        float peak = 0.f;
#pragma unroll 4
        for (int i = first; i < p.width; i += stride) {
            const Lanes<W> t = sum(i);
            if (p.residual) storeLanes<T, W>(static_cast<T *>(p.total) + row * p.width + i, t);
#pragma unroll
            for (int j = 0; j < W; ++j) peak = larger(peak, fabsf(t.at(j)));
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) peak = larger(peak, __shfl_xor_sync(0xffffffffu, peak, d));
        if (lane == 0) peaks[slot][threadIdx.x >> 5] = peak;
        __syncthreads();
        peak = peaks[slot][lane];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) peak = larger(peak, __shfl_xor_sync(0xffffffffu, peak, d));
        const float inverse = peak > 0.f ? 127.f / peak : 0.f;
        if (threadIdx.x == 0) p.scale[row] = peak / 127.f;
        int8_t *codes = p.codes + row * p.codesPitch;
#pragma unroll 4
        for (int i = first; i < p.width; i += stride) *reinterpret_cast<Pack<int8_t, W> *>(codes + i) = codesOf(sum(i), inverse);
        if (isinf(inverse)) tinyCodes<T, W>(p, row, 1.f, peak / 127.f, first, stride);
    }
}

struct NormGradient {
    int64_t rows;
    int width, team;
    Ring ring;
    const void *dy, *dtotal, *x, *residual, *weight;
    int64_t xPitch, residualPitch;
    const float *rms;
    int weightType;
    void *dx;
    float *partial;   // [CTAs][width], null where dweight is not wanted
};

// The sum is taken from x and residual again: from its rounded copy, dweight of a bfloat16 step would be off by 1.6e-3 in place of 1.6e-7.  A row is read twice, before and after
// its mean is known, from the ring.  Sums of dweight over a team's rows stay in registers, or in shared memory
// for 32 single elements a thread, where sums and weights would fill the registers (2000 x 16383 half 679 us with them there, 237 so; 1500 x 12001 in 32 bits 429 and 157).
template <int W, int ITEMS>
constexpr bool sumsInShared = W == 1 && ITEMS > 16;
// RINGED: arrays that come through the ring, 0, 4, or 3 for wide rows: dtotal is wanted last, so that it stays out of a ring that has no room for two stages of all four (4096 x 8192 in 32 bits 184
// us without a ring, 153 so; 2000 x 16384 half 151 and 102).
template <class T, int W, int ITEMS, int RINGED>
__global__ void __launch_bounds__(kMaxThreads, W * ITEMS <= 8 ? 2 : 1) addRmsNormGrad(const __grid_constant__ NormGradient p, int *status) {
    using Elements = Lanes<W>;
    __shared__ RingSpace space;
    __shared__ float sums[2][kMaxWarps];
    extern __shared__ __align__(16) uint8_t stages[];   // the ring; at the end [teams][width] sums of dweight
    float *teamPartial = reinterpret_cast<float *>(stages);
    const Team team(p.team);
    const int first = team.rank * W, stride = team.size * W, width = p.width;
    const float perElement = 1.f / static_cast<float>(width);
    if constexpr (RINGED > 0) space.init(p.ring.depth);
    waitForPredecessor();
    const int64_t step = static_cast<int64_t>(gridDim.x) * team.count, row0 = static_cast<int64_t>(blockIdx.x) * team.count;
    const Source sources[4] = {{p.dy, width}, {p.x, p.xPitch}, {p.residual, p.residualPitch}, {p.dtotal, width}};
    RingReader<T, RINGED> ring{sources, p.ring, p.rows, width, team.count, space.full, space.freed, stages};
    const int64_t rounds = row0 < p.rows ? (p.rows - row0 + step - 1) / step : 0;
    auto asks = [&](int64_t round) {   // the copies of a round, by the first warp
        if (threadIdx.x < 32 && round < rounds) ring.ask(row0 + round * step);
    };
    if constexpr (RINGED > 0)
        for (int i = 0; i < p.ring.depth; ++i) asks(i);
    float *mine = teamPartial + static_cast<size_t>(team.index) * width;
    auto weightOf = [&](int i) {
        Elements w = allOf<W>(0.f);
        if (first + i * stride < width)
#pragma unroll
            for (int j = 0; j < W; ++j) w.set(j, weightAt(p.weight, p.weightType, first + i * stride + j));
        return w;
    };
    constexpr bool kSumsInShared = sumsInShared<W, ITEMS>;
    static_assert(!kSumsInShared || RINGED == 0, "the sums lie where a ring would");
    constexpr int kBatch = 8;   // elements whose loads from memory are under way together; none of them passes a store, which might be to the same place
    Elements kept[kSumsInShared ? 1 : ITEMS], dw[kSumsInShared ? 1 : ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if constexpr (kSumsInShared) {
            if (first + i * stride < width) mine[first + i * stride] = 0.f;
        } else {
            kept[i] = weightOf(i);
            dw[i] = allOf<W>(0.f);
        }
    }
    letDependentsStart();
    bool alive = true;
    float rmsNext = rounds > 0 ? p.rms[min(row0 + team.index, p.rows - 1)] : 0.f;
    for (int64_t round = 0; round < rounds; ++round) {
        const int64_t first0 = row0 + round * step, row = first0 + team.index;
        const float rms = rmsNext;
        rmsNext = p.rms[min(row + step, p.rows - 1)];
        const T *dy = static_cast<const T *>(p.dy) + row * width, *dt = static_cast<const T *>(p.dtotal) + row * width;
        const T *x = static_cast<const T *>(p.x) + row * p.xPitch, *r = static_cast<const T *>(p.residual) + row * p.residualPitch;
        if constexpr (RINGED > 0) {
            if (alive) alive = ring.wait();
            if (round > 0) asks(round - 1 + p.ring.depth);   // into the stage of the round before, which all warps have read or are about to
            dy = ring.template row<(W > 1)>(0, first0, team.index);
            x = ring.template row<(W > 1)>(1, first0, team.index);
            r = ring.template row<(W > 1)>(2, first0, team.index);
            if constexpr (RINGED == 4) dt = ring.template row<(W > 1)>(3, first0, team.index);
        }
        const int here = row < p.rows ? width : 0;   // a row past the end adds nothing
        auto unit = [&](int at) {   // (x + residual) rms
            Elements t = loadLanes<T, W>(x + at);
            if (p.residual) t = t + loadLanes<T, W>(r + at);
            return t * rms;
        };
        // dy, (x + residual) rms and the weight of elements that a thread has one behind the other; the loads of an array together, without a branch between them
        auto batch = [&](int i0, float(&g)[kBatch], float(&u)[kBatch], float(&w)[kBatch]) {
            int at[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) at[i] = min(first + (i0 + i) * stride, width - 1);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                g[i] = toFloat(dy[at[i]]);
                u[i] = toFloat(x[at[i]]);
            }
            if (p.residual)
#pragma unroll
                for (int i = 0; i < kBatch; ++i) u[i] += toFloat(r[at[i]]);
            auto weights = [&](auto *from) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) w[i] = toFloat(from[at[i]]);
            };
            if (p.weightType == RXMET_TYPE_F32) weights(static_cast<const float *>(p.weight));
            else if (p.weightType == RXMET_TYPE_BF16) weights(static_cast<const __nv_bfloat16 *>(p.weight));
            else weights(static_cast<const __half *>(p.weight));
#pragma unroll
            for (int i = 0; i < kBatch; ++i) u[i] *= rms;
        };
        Elements dots = allOf<W>(0.f);
        if constexpr (kSumsInShared) {
#pragma unroll 1
            for (int i0 = 0; i0 < ITEMS; i0 += kBatch) {
                float g[kBatch], u[kBatch], w[kBatch];
                batch(i0, g, u, w);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int at = first + (i0 + i) * stride;
                    if (at >= here) continue;
                    dots.v = fmaf(g[i] * w[i], u[i], dots.v);
                    mine[at] = fmaf(g[i], u[i], mine[at]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int at = first + i * stride;
                if (at >= here) continue;
                const Elements g = loadLanes<T, W>(dy + at), u = unit(at);
                dots = dots.plus(g * kept[i], u);
                dw[i] = dw[i].plus(g, u);
            }
        }
        const float mean = team.sum(dots.total(), sums, round & 1) * perElement;
        T *dx = static_cast<T *>(p.dx) + row * width;
        auto gradient = [&](int at, const Elements &w) {
            Elements out = p.dtotal ? loadLanes<T, W>(dt + at) : allOf<W>(0.f);
            return out.plus((loadLanes<T, W>(dy + at) * w).plus(unit(at), -mean), rms);
        };
        if constexpr (kSumsInShared) {
#pragma unroll 1
            for (int i0 = 0; i0 < ITEMS; i0 += kBatch) {
                float g[kBatch], u[kBatch], w[kBatch], t[kBatch] = {};
                batch(i0, g, u, w);
                if (p.dtotal)
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) t[i] = toFloat(dt[min(first + (i0 + i) * stride, width - 1)]);
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (first + (i0 + i) * stride < here) dx[first + (i0 + i) * stride] = fromFloat<T>(fmaf(fmaf(g[i], w[i], u[i] * -mean), rms, t[i]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (first + i * stride < here) storeLanes<T, W>(dx + first + i * stride, gradient(first + i * stride, kept[i]));
        }
        if constexpr (RINGED > 0) ring.done();
    }
    if (!alive && (threadIdx.x & 31) == 0) atomicExch(status, 1);
    if (!p.partial) return;
    __syncthreads();   // the ring is read
    if constexpr (!kSumsInShared)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (first + i * stride < width) mine[first + i * stride + j] = dw[i].at(j);
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
        float s = 0.f;
        for (int k = 0; k < team.count; ++k) s += teamPartial[static_cast<size_t>(k) * width + c];
        p.partial[static_cast<size_t>(blockIdx.x) * width + c] = s;
    }
}

// dweight[c] = sum of the CTAs' parts: a CTA takes 32 columns, its warps every 32nd part.
__global__ void __launch_bounds__(1024) addRmsNormWeightGrad(const float *partial, int parts, int width, void *dweight, int type) {
    __shared__ float sums[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
    waitForPredecessor();
    float s = 0.f;
    if (c < width)
#pragma unroll 4
        for (int k = warp; k < parts; k += 32) s += partial[static_cast<size_t>(k) * width + c];
    sums[warp][threadIdx.x & 31] = s;
    __syncthreads();
    if (warp > 0 || c >= width) return;
    s = 0.f;
    for (int k = 0; k < 32; ++k) s += sums[k][threadIdx.x];
    if (type == RXMET_TYPE_F32) static_cast<float *>(dweight)[c] = s;
    else if (type == RXMET_TYPE_BF16) static_cast<__nv_bfloat16 *>(dweight)[c] = fromFloat<__nv_bfloat16>(s);
    else static_cast<__half *>(dweight)[c] = fromFloat<__half>(s);
}

struct TeamPlan {
    int team, threads;
    int teams() const { return threads / team; }
};
// The threads that a row needs at `perThread` elements each; CTAs of about 256.
TeamPlan teamFor(int width, int perThread) {
    const int needed = (width + perThread - 1) / perThread;
    int team = 8;
    while (team < needed && team < 32) team *= 2;
    if (needed > 32) team = (needed + 31) / 32 * 32;
    return {team, team * std::max(1, 256 / team)};
}

// f(W, ITEMS) as compile-time constants.  16-byte groups where every array's rows start on 16 bytes and the width is made of them, else single elements.  A thread takes
// sixteen elements, 32 of the widest rows and, in 16-byte groups, in front of codes: sums over a team cost the same for few as for many, and codes need two (8192 x 4096 bfloat16 with
// codes 8 elements 77 us, 16 60 us, 32 42 us; without 59, 49, 50, and 4096 x 8192 61 with 16 and 49 with 32, in 32 bits 84 and 94; gradients 92, 78, 93).  Half of them or a quarter where the rows are few and a row's latency counts (one row of
// 1024: 2.8 us, with 16 elements 3.8), or where 16 would leave lanes of a warp without any; four or twelve for gradients of single elements, whose registers 16 overflow (5003 x 1001
// 40 us for 34, 3000 x 5001 91 for 72).
enum class Output { Rows, Codes, Gradients };
template <class T, class F>
void withGroups(int64_t rows, int width, bool vector, Output output, F f) {
    constexpr int V = 16 / sizeof(T);
    const bool small = rows <= currentDevice().sms || width < 512;
    auto fits = [&](int perThread) { return width <= kMaxThreads * perThread; };
    using One = std::integral_constant<int, 1>;
    using VW = std::integral_constant<int, V>;
    if (vector) {
        if (small && fits(V)) return f(VW{}, One{});
        const bool wide = output == Output::Codes ? width >= 512 : output == Output::Rows && sizeof(T) == 2 && width > 256 * 16;
        if (fits(16) && !wide) return f(VW{}, std::integral_constant<int, 16 / V>{});
        return f(VW{}, std::integral_constant<int, 32 / V>{});
    }
    const bool gradients = output == Output::Gradients;
    if ((small || gradients) && fits(4)) return f(One{}, std::integral_constant<int, 4>{});
    if (gradients && fits(12)) return f(One{}, std::integral_constant<int, 12>{});
    if (fits(16)) return f(One{}, std::integral_constant<int, 16>{});
    return f(One{}, std::integral_constant<int, 32>{});
}

// A ring of two to four stages for as many CTAs as an SM's registers and shared memory hold; none where not even one has room for two.
Ring ringFor(const void *kernel, int width, size_t elementBytes, int arrays, const TeamPlan &plan) {
    constexpr size_t kAll = 224 * 1024;
    Ring ring;
    ring.arrayBytes = static_cast<uint32_t>(plan.teams() * (alignUp(width * elementBytes, 16) + 16) + 16);
    const size_t stage = static_cast<size_t>(ring.arrayBytes) * arrays;
    for (int ctas = residentPerSm(kernel, plan.threads, 0); ctas > 0; --ctas) {
        const size_t depth = (kAll / ctas - 1024) / stage;
        if (depth < 2) continue;
        ring.depth = static_cast<int>(std::min<size_t>(depth, Ring::kMaxDepth));
        return ring;
    }
    return {};
}

int gridFor(const void *kernel, int64_t rows, int teams, int threads, size_t smem) {
    const int64_t most = static_cast<int64_t>(currentDevice().sms) * residentPerSm(kernel, threads, smem);
    return static_cast<int>(std::max<int64_t>(1, std::min(most, (rows + teams - 1) / teams)));
}

void checkRows(int64_t rows, int width, int type, int weightType, int most = kMaxWidth) {
    RXMET_REQUIRE(rows >= 0 && width >= 1, "add_rms_norm: %lld rows of %d", static_cast<long long>(rows), width);
    if (width > most) fail(RXMET_ERR_UNSUPPORTED, "add_rms_norm: rows of %d elements, at most %d", width, most);
    RXMET_REQUIRE(type >= 0 && type <= 2 && weightType >= 0 && weightType <= 2, "add_rms_norm: unknown element type");
}

// Whether all rows start on 16 bytes, those of codes on as many as 16 bytes of T have elements, and consist of such groups.
template <bool Codes>
bool inGroups(const NormRows &p, int64_t group) {
    return p.width % group == 0 && p.xPitch % group == 0 && alignedTo(p.x, 16) &&
           (!p.residual || (p.residualPitch % group == 0 && alignedTo(p.residual, 16) && alignedTo(p.total, 16))) &&
           (Codes ? p.codesPitch % group == 0 && alignedTo(p.codes, group) : alignedTo(p.y, 16));
}

void launchWideCodes(const NormRows &p, int type, cudaStream_t st) {
    if (p.rows == 0) return;
    withType(type, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / sizeof(T);
        const auto kernel = inGroups<true>(p, V) ? codeWideRows<T, V> : codeWideRows<T, 1>;
        const int grid = gridFor(reinterpret_cast<const void *>(kernel), p.rows, 1, kWideThreads, 0);
        {
            KernelTimer timer__("codeWideRows", st);
            launchDependent(kernel, grid, kWideThreads, 0, st, p);
        }
        afterLaunch("codeWideRows");
    });
}

template <bool Codes>
void launchNorm(const char *name, NormRows p, int type, cudaStream_t st) {
    if (p.rows == 0) return;
    withType(type, [&](auto t) {
        using T = decltype(t);
        const bool vector = inGroups<Codes>(p, 16 / sizeof(T));
        withGroups<T>(p.rows, p.width, vector, Codes ? Output::Codes : Output::Rows, [&](auto w, auto items) {
            constexpr int W = decltype(w)::value, ITEMS = decltype(items)::value;
            const TeamPlan plan = teamFor(p.width, W * ITEMS);
            p.team = plan.team;
            // Rows that all fit the GPU's teams at once have no next ones to fetch, and a ring would only lengthen the way.
            if (p.rows > static_cast<int64_t>(currentDevice().sms) * plan.teams()) p.ring = ringFor(reinterpret_cast<const void *>(addRmsNorm<T, W, ITEMS, Codes, true>), p.width, sizeof(T), 2, plan);
            const auto kernel = p.ring.depth > 0 ? addRmsNorm<T, W, ITEMS, Codes, true> : addRmsNorm<T, W, ITEMS, Codes, false>;
            const size_t smem = static_cast<size_t>(p.ring.depth) * p.ring.arrayBytes * 2;
            ensureDynamicSmem(reinterpret_cast<const void *>(kernel), smem);
            const int grid = gridFor(reinterpret_cast<const void *>(kernel), p.rows, plan.teams(), plan.threads, smem);
            {
                KernelTimer timer__(name, st);
                launchDependent(kernel, grid, plan.threads, smem, st, p, waitStatus());
            }
            afterLaunch(name);
        });
    });
}

// CTAs of the gradient: those that are resident, but with some rows each, because a part of dweight is written for every one of them.
constexpr int kGradRowsOfTeam = 4;
template <class F>
void withGradKernel(int64_t rows, int width, int type, bool vector, F f) {
    withType(type, [&](auto t) {
        using T = decltype(t);
        withGroups<T>(rows, width, vector, Output::Gradients, [&](auto w, auto items) {
            constexpr int W = decltype(w)::value, ITEMS = decltype(items)::value;
            const TeamPlan plan = teamFor(width, W * ITEMS);
            const size_t partial = static_cast<size_t>(plan.teams()) * width * sizeof(float);
            // 64 bytes a thread are rows of up to 32 KB, of which a ring holds four or three arrays; longer ones have three, or no ring.
            constexpr int kBytes = W * ITEMS * static_cast<int>(sizeof(T));
            constexpr bool kRing = !sumsInShared<W, ITEMS>;
            Ring ring;
            void (*kernel)(NormGradient, int *) = nullptr;
            int arrays = 0;
            auto through = [&](auto count) {
                constexpr int ARRAYS = decltype(count)::value;
                if (kernel) return;
                if constexpr (ARRAYS > 0) {
                    ring = ringFor(reinterpret_cast<const void *>(addRmsNormGrad<T, W, ITEMS, ARRAYS>), width, sizeof(T), ARRAYS, plan);
                    if (ring.depth == 0) return;
                }
                kernel = addRmsNormGrad<T, W, ITEMS, ARRAYS>;
                arrays = ARRAYS;
            };
            if constexpr (kRing && kBytes <= 64) through(std::integral_constant<int, 4>{});
            if constexpr (kRing && kBytes >= 64) through(std::integral_constant<int, 3>{});
            if constexpr (!kRing || kBytes > 64) through(std::integral_constant<int, 0>{});
            if (!kernel) fail(RXMET_ERR_CUDA, "add_rms_norm backward: no kernel for rows of %d elements", width);
            const size_t smem = std::max(partial, static_cast<size_t>(ring.depth) * ring.arrayBytes * arrays);
            ensureDynamicSmem(reinterpret_cast<const void *>(kernel), smem);
            const int grid = gridFor(reinterpret_cast<const void *>(kernel), (rows + kGradRowsOfTeam - 1) / kGradRowsOfTeam, plan.teams(), plan.threads, smem);
            f(kernel, plan, ring, smem, grid);
        });
    });
}

}  // namespace
}  // namespace rxmet

using namespace rxmet;

extern "C" {

int rxmet_add_rms_norm(int64_t rows, int width, int type, const void *x_dev, int64_t x_pitch, const void *residual_dev,
                       int64_t residual_pitch, const void *weight_dev, int weight_type, float eps, void *total_dev, void *y_dev,
                       float *rms_dev, void *stream) {
    return guarded([&] {
        checkRows(rows, width, type, weight_type);
        RXMET_REQUIRE(rows == 0 || (x_dev && weight_dev && y_dev && (!residual_dev || total_dev)), "add_rms_norm: null tensor");
        NormRows p{rows, width, 1, {}, x_dev, residual_dev, weight_dev, x_pitch, residual_pitch, weight_type, eps, total_dev, y_dev, rms_dev, nullptr, 0, nullptr};
        launchNorm<false>("addRmsNorm", p, type, static_cast<cudaStream_t>(stream));
    });
}

int rxmet_add_rms_norm_codes(int64_t rows, int width, int type, const void *x_dev, int64_t x_pitch, const void *residual_dev,
                             int64_t residual_pitch, const void *weight_dev, int weight_type, float eps, void *total_dev,
                             int8_t *codes_dev, int64_t codes_pitch, float *scale_dev, void *stream) {
    return guarded([&] {
        checkRows(rows, width, type, weight_type, weight_dev ? kMaxWidth : kMaxCoded);
        RXMET_REQUIRE(rows == 0 || (x_dev && codes_dev && scale_dev && (!residual_dev || total_dev)), "add_rms_norm_codes: null tensor");
        RXMET_REQUIRE(codes_pitch >= width, "add_rms_norm_codes: rows of %d codes %lld bytes apart", width, static_cast<long long>(codes_pitch));
        NormRows p{rows, width, 1, {}, x_dev, residual_dev, weight_dev, x_pitch, residual_pitch, weight_type, eps, total_dev, nullptr, nullptr, codes_dev, codes_pitch, scale_dev};
        if (width > kMaxWidth) launchWideCodes(p, type, static_cast<cudaStream_t>(stream));
        else launchNorm<true>("addRmsNormCodes", p, type, static_cast<cudaStream_t>(stream));
    });
}

size_t rxmet_add_rms_norm_backward_workspace_bytes(int64_t rows, int width, int type) {
    size_t bytes = 0;
    guarded([&] {
        checkRows(rows, width, type, RXMET_TYPE_F32);
        for (const bool vector : {false, true})
            withGradKernel(rows, width, type, vector, [&](auto, TeamPlan, Ring, size_t, int grid) {
                bytes = std::max(bytes, static_cast<size_t>(grid) * width * sizeof(float));
            });
    });
    return bytes;
}

int rxmet_add_rms_norm_backward(int64_t rows, int width, int type, const void *dy_dev, const void *dtotal_dev, const void *x_dev,
                                int64_t x_pitch, const void *residual_dev, int64_t residual_pitch, const float *rms_dev, const void *weight_dev, int weight_type, void *dx_dev,
                                void *dweight_dev, void *workspace_dev, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        checkRows(rows, width, type, weight_type);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (rows == 0) {
            if (dweight_dev) RXMET_CUDA(cudaMemsetAsync(dweight_dev, 0, width * typeBytes(weight_type), st));
            return;
        }
        RXMET_REQUIRE(dy_dev && x_dev && rms_dev && weight_dev && dx_dev, "add_rms_norm backward: null tensor");
        const int64_t group = 16 / static_cast<int64_t>(typeBytes(type));
        const bool vector = width % group == 0 && x_pitch % group == 0 && residual_pitch % group == 0 && alignedTo(dy_dev, 16) && alignedTo(dtotal_dev, 16) &&
                            alignedTo(x_dev, 16) && alignedTo(residual_dev, 16) && alignedTo(dx_dev, 16);
        withGradKernel(rows, width, type, vector, [&](auto kernel, TeamPlan plan, Ring ring, size_t smem, int grid) {
            NormGradient p{rows, width, plan.team, ring, dy_dev, dtotal_dev, x_dev, residual_dev, weight_dev, x_pitch, residual_pitch, rms_dev, weight_type, dx_dev, nullptr};
            if (dweight_dev) p.partial = Workspace(workspace_dev, workspace_bytes).take<float>(static_cast<size_t>(grid) * width);
            {
                KernelTimer timer__("addRmsNormGrad", st);
                launchDependent(kernel, grid, plan.threads, smem, st, p, waitStatus());
            }
            afterLaunch("addRmsNormGrad");
            if (!dweight_dev) return;
            {
                KernelTimer timer__("addRmsNormWeightGrad", st);
                launchDependent(addRmsNormWeightGrad, (width + 31) / 32, 1024, 0, st, static_cast<const float *>(p.partial), grid, width, dweight_dev, weight_type);
            }
            afterLaunch("addRmsNormWeightGrad");
        });
    });
}

}  // extern "C"
