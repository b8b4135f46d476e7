// Residual addition with a root-mean-square norm (to the input's type, or to 8-bit codes with a scale for each row), and its gradient.
//
// One pass over the data: a team of 8 to 512 threads holds a row in registers, so that the sum, the largest magnitude and the output need no
// second read.  A team walks over rows, which keeps the weights in registers, and asks for its next row before it works on this one.
// Sums run in 32 bits: a thread's own elements in order, lanes as a tree, warps in order, so that results do not depend on the grid.
//
// Bound: HBM.
#include <algorithm>

#include "common.h"
#include "dependent_launch.cuh"
#include "element_types.cuh"

namespace rxmet {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kMaxThreads = 512, kMaxWarps = kMaxThreads / 32;

struct NormRows {
    int64_t rows;
    int width, team;   // team: its threads, a power of two up to 32 or a multiple of it
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

// The place of a thread in its team.  Teams of a CTA work on rows of their own; those of several warps meet at a barrier of their own.
struct Team {
    int size, index, count, rank;
    __device__ __forceinline__ explicit Team(int threads) : size(threads), index(threadIdx.x / threads), count(blockDim.x / threads), rank(threadIdx.x - index * threads) {}
    template <class V>
    __device__ __forceinline__ void meet(V (*shared)[kMaxWarps], int slot, V mine) const {
        if ((threadIdx.x & 31) == 0) shared[slot][threadIdx.x >> 5] = mine;
        asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(size) : "memory");
    }
    // `slot` alternates between two arrays from row to row, so that one barrier is enough.
    __device__ __forceinline__ float sum(float v, float (*shared)[kMaxWarps], int slot) const {
        for (int d = min(size, 32) / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (size <= 32) return v;
        meet(shared, slot, v);
        const int first = index * size / 32;
        v = 0.f;
        for (int i = 0; i < size / 32; ++i) v += shared[slot][first + i];
        return v;
    }
    // Largest magnitude as bits: patterns of non-negative floats order as integers, with NaN above infinity, so that a NaN is not lost.
    __device__ __forceinline__ uint32_t most(uint32_t v, uint32_t (*shared)[kMaxWarps], int slot) const {
        for (int d = min(size, 32) / 2; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
        if (size <= 32) return v;
        meet(shared, slot, v);
        const int first = index * size / 32;
        v = 0;
        for (int i = 0; i < size / 32; ++i) v = max(v, shared[slot][first + i]);
        return v;
    }
};

__device__ __forceinline__ float weightAt(const void *weight, int type, int i) {
    if (type == RXMET_TYPE_F32) return static_cast<const float *>(weight)[i];
    if (type == RXMET_TYPE_BF16) return toFloat(static_cast<const __nv_bfloat16 *>(weight)[i]);
    return toFloat(static_cast<const __half *>(weight)[i]);
}

// A thread's share of a row: ITEMS groups of W neighbouring elements, `stride` elements apart; what lies beyond the row is zero.
template <class T, int W, int ITEMS>
struct Share {
    Pack<T, W> v[ITEMS];
    __device__ __forceinline__ void load(const T *row, int first, int stride, int width) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            v[i] = {};
            if (first + i * stride < width) v[i] = *reinterpret_cast<const Pack<T, W> *>(row + first + i * stride);
        }
    }
    __device__ __forceinline__ float at(int i, int j) const { return toFloat(v[i].v[j]); }
};
template <class T, int W>
__device__ __forceinline__ void put(T *row, int at, const float (&v)[W]) {
    Pack<T, W> out;
#pragma unroll
    for (int j = 0; j < W; ++j) out.v[j] = fromFloat<T>(v[j]);
    *reinterpret_cast<Pack<T, W> *>(row + at) = out;
}

// Up to 16 elements a thread, the next row is in registers before this one is done and the weights stay there; wider rows have a thread's own loads to cover one another,
// and read the weights again.
template <int W, int ITEMS>
constexpr bool kAhead = W *ITEMS <= 16;

template <class T, int W, int ITEMS, bool Codes>
__global__ void __launch_bounds__(kMaxThreads) addRmsNorm(const __grid_constant__ NormRows p) {
    constexpr bool Ahead = kAhead<W, ITEMS>;
    __shared__ float sums[2][kMaxWarps];
    __shared__ uint32_t peaks[2][kMaxWarps];
    const Team team(p.team);
    const int first = team.rank * W, stride = team.size * W, width = p.width;
    const bool norm = p.weight != nullptr;
    waitForPredecessor();
    const int64_t step = static_cast<int64_t>(gridDim.x) * team.count;
    int64_t row = static_cast<int64_t>(blockIdx.x) * team.count + team.index;
    Share<T, W, ITEMS> x, r;
    auto ask = [&](int64_t at) {
        at = min(at, p.rows - 1);   // past the end: a row that is there, and dropped
        x.load(static_cast<const T *>(p.x) + at * p.xPitch, first, stride, width);
        if (p.residual) r.load(static_cast<const T *>(p.residual) + at * p.residualPitch, first, stride, width);
    };
    ask(row);
    float w[Ahead ? ITEMS : 1][W];
    auto weights = [&](float(&to)[W], int i) {
#pragma unroll
        for (int j = 0; j < W; ++j) to[j] = norm && first + i * stride < width ? weightAt(p.weight, p.weightType, first + i * stride + j) : 1.f;
    };
    if constexpr (Ahead)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) weights(w[i], i);
    letDependentsStart();
    // all teams of a warp go through the same number of rows, because they shuffle together
    const int64_t rounds = (p.rows + step - 1) / step;
    for (int64_t round = 0; round < rounds; ++round, row += step) {
        const int slot = round & 1;
        const bool real = row < p.rows;
        float t[ITEMS][W], sum = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                t[i][j] = p.residual ? x.at(i, j) + r.at(i, j) : x.at(i, j);
                sum = fmaf(t[i][j], t[i][j], sum);
            }
        if (Ahead && round + 1 < rounds) ask(row + step);
        if (p.residual && real) {
            T *total = static_cast<T *>(p.total) + row * width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (first + i * stride < width) put(total, first + i * stride, t[i]);
        }
        float rms = 1.f;
        if (norm) {
            rms = rsqrtf(team.sum(sum, sums, slot) / static_cast<float>(width) + p.eps);
            if (p.rms && first == 0 && real) p.rms[row] = rms;
        }
        uint32_t peak = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if constexpr (!Ahead) weights(w[0], i);
            const bool in = first + i * stride < width;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                t[i][j] = t[i][j] * rms * w[Ahead ? i : 0][j];
                if (Codes && in) peak = max(peak, __float_as_uint(t[i][j]) & 0x7fffffffu);
            }
        }
        if constexpr (Codes) {
            const float most = __uint_as_float(team.most(peak, peaks, slot));
            const float inverse = most > 0.f ? 127.f / most : 0.f;
            if (real) {
                if (first == 0) p.scale[row] = most / 127.f;
                int8_t *codes = p.codes + row * p.codesPitch;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    Pack<int8_t, W> out;
#pragma unroll
                    for (int j = 0; j < W; ++j) out.v[j] = static_cast<int8_t>(__float2int_rn(fminf(fmaxf(t[i][j] * inverse, -127.f), 127.f)));
                    if (first + i * stride < width) *reinterpret_cast<Pack<int8_t, W> *>(codes + first + i * stride) = out;
                }
            }
        } else if (real) {
            T *y = static_cast<T *>(p.y) + row * width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (first + i * stride < width) put(y, first + i * stride, t[i]);
        }
        if (!Ahead && round + 1 < rounds) ask(row + step);
    }
}

struct NormGradient {
    int64_t rows;
    int width, team;
    const void *dy, *dtotal, *x, *residual, *weight;
    int64_t xPitch, residualPitch;
    const float *rms;
    int weightType;
    void *dx;
    float *partial;   // [CTAs][width], null where dweight is not wanted
};

// The sum is taken from x and residual again: from its rounded copy, dweight of a bfloat16 step would be off by 1.6e-3 in place of 1.6e-7.  Sums of dweight over a team's
// rows stay in registers, of wide rows in shared memory, where each element has one thread.
template <class T, int W, int ITEMS>
__global__ void __launch_bounds__(kMaxThreads) addRmsNormGrad(const __grid_constant__ NormGradient p) {
    constexpr bool Ahead = kAhead<W, ITEMS>;
    __shared__ float sums[2][kMaxWarps];
    extern __shared__ float teamPartial[];   // [teams][width]
    const Team team(p.team);
    const int first = team.rank * W, stride = team.size * W, width = p.width;
    waitForPredecessor();
    const int64_t step = static_cast<int64_t>(gridDim.x) * team.count;
    int64_t row = static_cast<int64_t>(blockIdx.x) * team.count + team.index;
    Share<T, W, ITEMS> dy, dt, x, r;
    float rmsNext = 0.f;
    auto ask = [&](int64_t at) {
        const bool real = at < p.rows;
        at = min(at, p.rows - 1);
        dy.load(static_cast<const T *>(p.dy) + at * width, first, stride, real ? width : 0);   // a row past the end adds nothing
        x.load(static_cast<const T *>(p.x) + at * p.xPitch, first, stride, width);
        if (p.residual) r.load(static_cast<const T *>(p.residual) + at * p.residualPitch, first, stride, width);
        if (p.dtotal) dt.load(static_cast<const T *>(p.dtotal) + at * width, first, stride, width);
        rmsNext = p.rms[at];
    };
    ask(row);
    float *mine = teamPartial + static_cast<size_t>(team.index) * width;
    float w[Ahead ? ITEMS : 1][W], dw[Ahead ? ITEMS : 1][W];
    auto weights = [&](float(&to)[W], int i) {
#pragma unroll
        for (int j = 0; j < W; ++j) to[j] = first + i * stride < width ? weightAt(p.weight, p.weightType, first + i * stride + j) : 0.f;
    };
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if constexpr (Ahead) {
            weights(w[i], i);
#pragma unroll
            for (int j = 0; j < W; ++j) dw[i][j] = 0.f;
        } else if (p.partial && first + i * stride < width) {
#pragma unroll
            for (int j = 0; j < W; ++j) mine[first + i * stride + j] = 0.f;
        }
    }
    letDependentsStart();
    const int64_t rounds = (p.rows + step - 1) / step;
    for (int64_t round = 0; round < rounds; ++round, row += step) {
        const float rms = rmsNext;
        float u[ITEMS][W], sum = 0.f;
        const Share<T, W, ITEMS> g = dy, add = dt;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if constexpr (!Ahead) weights(w[0], i);
            const bool in = first + i * stride < width;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                u[i][j] = (p.residual ? x.at(i, j) + r.at(i, j) : x.at(i, j)) * rms;
                sum = fmaf(g.at(i, j) * w[Ahead ? i : 0][j], u[i][j], sum);
                if constexpr (Ahead) dw[i][j] = fmaf(g.at(i, j), u[i][j], dw[i][j]);
                else if (p.partial && in) mine[first + i * stride + j] = fmaf(g.at(i, j), u[i][j], mine[first + i * stride + j]);
            }
        }
        if (Ahead && round + 1 < rounds) ask(row + step);
        const float mean = team.sum(sum, sums, round & 1) / static_cast<float>(width);
        if (row < p.rows) {
            T *dx = static_cast<T *>(p.dx) + row * width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                if (first + i * stride >= width) continue;
                if constexpr (!Ahead) weights(w[0], i);
                float out[W];
#pragma unroll
                for (int j = 0; j < W; ++j) out[j] = fmaf(rms, fmaf(-u[i][j], mean, g.at(i, j) * w[Ahead ? i : 0][j]), p.dtotal ? add.at(i, j) : 0.f);
                put(dx, first + i * stride, out);
            }
        }
        if (!Ahead && round + 1 < rounds) ask(row + step);
    }
    if (!p.partial) return;
    if constexpr (Ahead)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (first + i * stride < width) mine[first + i * stride + j] = dw[i][j];
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

// f(W, ITEMS) as compile-time constants.  16-byte groups where every array's rows start on 16 bytes and the width is made of them, else single elements; the fewest groups a
// thread with which a team holds the row.
template <class T, class F>
void withGroups(int width, bool vector, F f) {
    constexpr int V = 16 / sizeof(T);
    auto fits = [&](int perThread) { return width <= kMaxThreads * perThread; };
    auto run = [&](auto w, auto items) { return f(w, items); };
    using One = std::integral_constant<int, 1>;
    using VW = std::integral_constant<int, V>;
    if (vector) {
        if (fits(V)) return run(VW{}, One{});
        if (fits(2 * V)) return run(VW{}, std::integral_constant<int, 2>{});
        return run(VW{}, std::integral_constant<int, 32 / V>{});
    }
    if (fits(4)) return run(One{}, std::integral_constant<int, 4>{});
    if (fits(16)) return run(One{}, std::integral_constant<int, 16>{});
    return run(One{}, std::integral_constant<int, 32>{});
}

int gridFor(const void *kernel, int64_t rows, int teams, int threads, size_t smem) {
    const int64_t most = static_cast<int64_t>(currentDevice().sms) * residentPerSm(kernel, threads, smem);
    return static_cast<int>(std::max<int64_t>(1, std::min(most, (rows + teams - 1) / teams)));
}

void checkRows(int64_t rows, int width, int type, int weightType) {
    RXMET_REQUIRE(rows >= 0 && width >= 1, "add_rms_norm: %lld rows of %d", static_cast<long long>(rows), width);
    if (width > kMaxWidth) fail(RXMET_ERR_UNSUPPORTED, "add_rms_norm: rows of %d elements, at most %d", width, kMaxWidth);
    RXMET_REQUIRE(type >= 0 && type <= 2 && weightType >= 0 && weightType <= 2, "add_rms_norm: unknown element type");
}

template <bool Codes>
void launchNorm(const char *name, NormRows p, int type, cudaStream_t st) {
    if (p.rows == 0) return;
    withType(type, [&](auto t) {
        using T = decltype(t);
        const int64_t group = 16 / sizeof(T);
        const bool vector = p.width % group == 0 && p.xPitch % group == 0 && alignedTo(p.x, 16) &&
                            (!p.residual || (p.residualPitch % group == 0 && alignedTo(p.residual, 16) && alignedTo(p.total, 16))) &&
                            (Codes ? p.codesPitch % group == 0 && alignedTo(p.codes, group) : alignedTo(p.y, 16));
        withGroups<T>(p.width, vector, [&](auto w, auto items) {
            constexpr int W = decltype(w)::value, ITEMS = decltype(items)::value;
            const auto kernel = addRmsNorm<T, W, ITEMS, Codes>;
            const TeamPlan plan = teamFor(p.width, W * ITEMS);
            p.team = plan.team;
            const int grid = gridFor(reinterpret_cast<const void *>(kernel), p.rows, plan.teams(), plan.threads, 0);
            {
                KernelTimer timer__(name, st);
                launchDependent(kernel, grid, plan.threads, 0, st, p);
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
        withGroups<T>(width, vector, [&](auto w, auto items) {
            constexpr int W = decltype(w)::value, ITEMS = decltype(items)::value;
            const auto kernel = addRmsNormGrad<T, W, ITEMS>;
            const TeamPlan plan = teamFor(width, W * ITEMS);
            const size_t smem = static_cast<size_t>(plan.teams()) * width * sizeof(float);
            ensureDynamicSmem(reinterpret_cast<const void *>(kernel), smem);
            const int grid = gridFor(reinterpret_cast<const void *>(kernel), (rows + kGradRowsOfTeam - 1) / kGradRowsOfTeam, plan.teams(), plan.threads, smem);
            f(kernel, plan, smem, grid);
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
        NormRows p{rows, width, 1, x_dev, residual_dev, weight_dev, x_pitch, residual_pitch, weight_type, eps, total_dev, y_dev, rms_dev, nullptr, 0, nullptr};
        launchNorm<false>("addRmsNorm", p, type, static_cast<cudaStream_t>(stream));
    });
}

int rxmet_add_rms_norm_codes(int64_t rows, int width, int type, const void *x_dev, int64_t x_pitch, const void *residual_dev,
                             int64_t residual_pitch, const void *weight_dev, int weight_type, float eps, void *total_dev,
                             int8_t *codes_dev, int64_t codes_pitch, float *scale_dev, void *stream) {
    return guarded([&] {
        checkRows(rows, width, type, weight_type);
        RXMET_REQUIRE(rows == 0 || (x_dev && codes_dev && scale_dev && (!residual_dev || total_dev)), "add_rms_norm_codes: null tensor");
        RXMET_REQUIRE(codes_pitch >= width, "add_rms_norm_codes: rows of %d codes %lld bytes apart", width, static_cast<long long>(codes_pitch));
        NormRows p{rows, width, 1, x_dev, residual_dev, weight_dev, x_pitch, residual_pitch, weight_type, eps, total_dev, nullptr, nullptr, codes_dev, codes_pitch, scale_dev};
        launchNorm<true>("addRmsNormCodes", p, type, static_cast<cudaStream_t>(stream));
    });
}

size_t rxmet_add_rms_norm_backward_workspace_bytes(int64_t rows, int width, int type) {
    size_t bytes = 0;
    guarded([&] {
        checkRows(rows, width, type, RXMET_TYPE_F32);
        for (const bool vector : {false, true})
            withGradKernel(rows, width, type, vector, [&](auto, TeamPlan, size_t, int grid) {
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
        withGradKernel(rows, width, type, vector, [&](auto kernel, TeamPlan plan, size_t smem, int grid) {
            NormGradient p{rows, width, plan.team, dy_dev, dtotal_dev, x_dev, residual_dev, weight_dev, x_pitch, residual_pitch, rms_dev, weight_type, dx_dev, nullptr};
            if (dweight_dev) p.partial = Workspace(workspace_dev, workspace_bytes).take<float>(static_cast<size_t>(grid) * width);
            {
                KernelTimer timer__("addRmsNormGrad", st);
                launchDependent(kernel, grid, plan.threads, smem, st, p);
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
