// Residual addition with a root-mean-square norm (to the input's type, or to 8-bit codes with a scale for each row), and its gradient.
//
// One pass over the data: a team of 1 to 32 warps holds a row in registers, so that the sum, the largest magnitude and the output need no
// second read.  A team walks over rows, which keeps the weights in registers, and asks for its next row before it works on this one.
// Sums run in 32 bits: a lane's own elements in order, lanes and warps as a fixed tree, so that results do not depend on the launch.
//
// Bound: HBM.
#include <algorithm>

#include "common.h"
#include "dependent_launch.cuh"
#include "element_types.cuh"

namespace rxmet {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kMaxWarps = 32;

struct NormRows {
    int64_t rows;
    int width, teamWarps;
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

__device__ __forceinline__ float warpSum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Sum over the warps of a team; `slot` alternates between two arrays from row to row, so that one barrier is enough.
__device__ __forceinline__ float teamSum(float v, int teamWarps, float (*shared)[kMaxWarps], int slot) {
    v = warpSum(v);
    if (teamWarps == 1) return v;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) shared[slot][warp] = v;
    __syncthreads();
    float sum = 0.f;
    for (int i = 0; i < teamWarps; ++i) sum += shared[slot][i];
    return sum;
}
// Largest magnitude as bits: patterns of non-negative floats order as integers, with NaN above infinity, so that a NaN is not lost.
__device__ __forceinline__ uint32_t teamMax(uint32_t v, int teamWarps, uint32_t (*shared)[kMaxWarps], int slot) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (teamWarps == 1) return v;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) shared[slot][warp] = v;
    __syncthreads();
    uint32_t most = 0;
    for (int i = 0; i < teamWarps; ++i) most = max(most, shared[slot][i]);
    return most;
}

__device__ __forceinline__ float weightAt(const void *weight, int type, int i) {
    if (type == RXMET_TYPE_F32) return static_cast<const float *>(weight)[i];
    if (type == RXMET_TYPE_BF16) return toFloat(static_cast<const __nv_bfloat16 *>(weight)[i]);
    return toFloat(static_cast<const __half *>(weight)[i]);
}

// A thread's share of a row: ITEMS groups of W neighbouring elements, `stride` elements apart.
template <class T, int W, int ITEMS>
struct Share {
    Pack<T, W> v[ITEMS];
    __device__ __forceinline__ void load(const T *row, int first, int stride, int width) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (first + i * stride < width) v[i] = *reinterpret_cast<const Pack<T, W> *>(row + first + i * stride);
    }
};

// Teams of a CTA work on rows of their own; only a CTA of one team (more than one warp) has barriers.
// THREADS: the most that a CTA may have, 512 or 1024.
template <class T, int W, int ITEMS, bool Codes, int THREADS>
__global__ void __launch_bounds__(THREADS) addRmsNorm(const __grid_constant__ NormRows p) {
    __shared__ float sums[2][kMaxWarps];
    __shared__ uint32_t peaks[2][kMaxWarps];
    const int teamThreads = p.teamWarps * 32, team = threadIdx.x / teamThreads, teams = blockDim.x / teamThreads;
    const int first = (threadIdx.x - team * teamThreads) * W, stride = teamThreads * W, width = p.width;
    const bool norm = p.weight != nullptr;
    waitForPredecessor();
    float w[ITEMS][W];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = norm && first + i * stride < width ? weightAt(p.weight, p.weightType, first + i * stride + j) : 1.f;

    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    int64_t row = static_cast<int64_t>(blockIdx.x) * teams + team;
    Share<T, W, ITEMS> x, r;
    auto ask = [&](int64_t at) {
        if (at >= p.rows) return;
        x.load(static_cast<const T *>(p.x) + at * p.xPitch, first, stride, width);
        if (p.residual) r.load(static_cast<const T *>(p.residual) + at * p.residualPitch, first, stride, width);
    };
    ask(row);
    letDependentsStart();
    for (int slot = 0; row < p.rows; row += step, slot ^= 1) {
        float t[ITEMS][W], sum = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const bool in = first + i * stride < width;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                t[i][j] = in ? toFloat(x.v[i].v[j]) + (p.residual ? toFloat(r.v[i].v[j]) : 0.f) : 0.f;
                sum = fmaf(t[i][j], t[i][j], sum);
            }
        }
        ask(row + step);
        if (p.residual) {
            T *total = static_cast<T *>(p.total) + row * width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                Pack<T, W> out;
#pragma unroll
                for (int j = 0; j < W; ++j) out.v[j] = fromFloat<T>(t[i][j]);
                if (first + i * stride < width) *reinterpret_cast<Pack<T, W> *>(total + first + i * stride) = out;
            }
        }
        float rms = 1.f;
        if (norm) {
            rms = rsqrtf(teamSum(sum, p.teamWarps, sums, slot) / static_cast<float>(width) + p.eps);
            if (p.rms && first == 0) p.rms[row] = rms;
        }
        uint32_t peak = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                t[i][j] = t[i][j] * rms * w[i][j];
                if (Codes && first + i * stride < width) peak = max(peak, __float_as_uint(t[i][j]) & 0x7fffffffu);
            }
        if constexpr (Codes) {
            const float most = __uint_as_float(teamMax(peak, p.teamWarps, peaks, slot));
            const float inverse = most > 0.f ? 127.f / most : 0.f;
            if (first == 0) p.scale[row] = most / 127.f;
            int8_t *codes = p.codes + row * p.codesPitch;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                Pack<int8_t, W> out;
#pragma unroll
                for (int j = 0; j < W; ++j) out.v[j] = static_cast<int8_t>(__float2int_rn(fminf(fmaxf(t[i][j] * inverse, -127.f), 127.f)));
                if (first + i * stride < width) *reinterpret_cast<Pack<int8_t, W> *>(codes + first + i * stride) = out;
            }
        } else {
            T *y = static_cast<T *>(p.y) + row * width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                Pack<T, W> out;
#pragma unroll
                for (int j = 0; j < W; ++j) out.v[j] = fromFloat<T>(t[i][j]);
                if (first + i * stride < width) *reinterpret_cast<Pack<T, W> *>(y + first + i * stride) = out;
            }
        }
    }
}

struct NormGradient {
    int64_t rows;
    int width, teamWarps;
    const void *dy, *dtotal, *x, *residual, *weight;
    int64_t xPitch, residualPitch;
    const float *rms;
    int weightType;
    void *dx;
    float *partial;   // [CTAs][width], null where dweight is not wanted
};

// The sum is taken from x and residual again: from its rounded copy, dweight of a bfloat16 step would be off by 1.6e-3 in place of 1.6e-7.
template <class T, int W, int ITEMS, int THREADS>
__global__ void __launch_bounds__(THREADS) addRmsNormGrad(const __grid_constant__ NormGradient p) {
    __shared__ float sums[2][kMaxWarps];
    extern __shared__ float teamPartial[];   // [teams][width] where a CTA has more than one team
    const int teamThreads = p.teamWarps * 32, team = threadIdx.x / teamThreads, teams = blockDim.x / teamThreads;
    const int first = (threadIdx.x - team * teamThreads) * W, stride = teamThreads * W, width = p.width;
    waitForPredecessor();
    float w[ITEMS][W], dw[ITEMS][W];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            w[i][j] = first + i * stride < width ? weightAt(p.weight, p.weightType, first + i * stride + j) : 0.f;
            dw[i][j] = 0.f;
        }
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    int64_t row = static_cast<int64_t>(blockIdx.x) * teams + team;
    Share<T, W, ITEMS> dy, dt, x, r;
    float rmsNext = 0.f;
    auto ask = [&](int64_t at) {
        if (at >= p.rows) return;
        dy.load(static_cast<const T *>(p.dy) + at * width, first, stride, width);
        x.load(static_cast<const T *>(p.x) + at * p.xPitch, first, stride, width);
        if (p.residual) r.load(static_cast<const T *>(p.residual) + at * p.residualPitch, first, stride, width);
        if (p.dtotal) dt.load(static_cast<const T *>(p.dtotal) + at * width, first, stride, width);
        rmsNext = p.rms[at];
    };
    ask(row);
    letDependentsStart();
    for (int slot = 0; row < p.rows; row += step, slot ^= 1) {
        const float rms = rmsNext;
        float u[ITEMS][W], d[ITEMS][W], add[ITEMS][W], sum = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const bool in = first + i * stride < width;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float g = in ? toFloat(dy.v[i].v[j]) : 0.f;
                u[i][j] = in ? (toFloat(x.v[i].v[j]) + (p.residual ? toFloat(r.v[i].v[j]) : 0.f)) * rms : 0.f;
                add[i][j] = in && p.dtotal ? toFloat(dt.v[i].v[j]) : 0.f;
                dw[i][j] = fmaf(g, u[i][j], dw[i][j]);
                d[i][j] = g * w[i][j];
                sum = fmaf(d[i][j], u[i][j], sum);
            }
        }
        ask(row + step);
        const float mean = teamSum(sum, p.teamWarps, sums, slot) / static_cast<float>(width);
        T *dx = static_cast<T *>(p.dx) + row * width;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            Pack<T, W> out;
#pragma unroll
            for (int j = 0; j < W; ++j) out.v[j] = fromFloat<T>(fmaf(rms, fmaf(-u[i][j], mean, d[i][j]), add[i][j]));
            if (first + i * stride < width) *reinterpret_cast<Pack<T, W> *>(dx + first + i * stride) = out;
        }
    }
    if (!p.partial) return;
    float *mine = teams == 1 ? p.partial + static_cast<size_t>(blockIdx.x) * width : teamPartial + static_cast<size_t>(team) * width;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (first + i * stride < width) mine[first + i * stride + j] = dw[i][j];
    if (teams == 1) return;
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
        float s = 0.f;
        for (int k = 0; k < teams; ++k) s += teamPartial[static_cast<size_t>(k) * width + c];
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
    int warps, threads;
};
// The smallest team (a power of two of warps) that holds a row at ITEMS groups of W elements a thread; narrow rows put four teams of one warp into a CTA.
TeamPlan teamFor(int width, int perThread) {
    int warps = 1;
    while (warps * 32 * perThread < width) warps *= 2;
    return {warps, warps == 1 ? 128 : warps * 32};
}

// f(W, ITEMS) as compile-time constants.  16-byte groups where every array's rows start on 16 bytes and the width is made of them, else single elements.
// `items`: groups a thread may hold.  Few rows take fewer groups a thread, because then the row's latency counts and not the warps that it takes.
template <class T, int MaxItems, class F>
void withGroups(int64_t rows, int width, bool vector, F f) {
    constexpr int V = 16 / sizeof(T);
    if (!vector) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
    using VW = std::integral_constant<int, V>;
    auto fits = [&](int items) { return width <= kMaxWarps * 32 * V * items; };
    const bool few = rows <= currentDevice().sms;
    if (fits(1) && (few || width <= 32 * V)) return f(VW{}, std::integral_constant<int, 1>{});
    if (fits(2) && (few || MaxItems == 2 || width <= 64 * V)) return f(VW{}, std::integral_constant<int, 2>{});
    return f(VW{}, std::integral_constant<int, 4>{});
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
        withGroups<T, 4>(p.rows, p.width, vector, [&](auto w, auto items) {
            constexpr int W = decltype(w)::value, ITEMS = decltype(items)::value;
            const TeamPlan plan = teamFor(p.width, W * ITEMS);
            const auto kernel = plan.threads > 512 ? addRmsNorm<T, W, ITEMS, Codes, 1024> : addRmsNorm<T, W, ITEMS, Codes, 512>;
            p.teamWarps = plan.warps;
            const int teams = plan.threads / (plan.warps * 32);
            const int grid = gridFor(reinterpret_cast<const void *>(kernel), p.rows, teams, plan.threads, 0);
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
        withGroups<T, 2>(rows, width, vector, [&](auto w, auto items) {
            constexpr int W = decltype(w)::value, ITEMS = decltype(items)::value;
            const TeamPlan plan = teamFor(width, W * ITEMS);
            const auto kernel = plan.threads > 512 ? addRmsNormGrad<T, W, ITEMS, 1024> : addRmsNormGrad<T, W, ITEMS, 512>;
            const int teams = plan.threads / (plan.warps * 32);
            const size_t smem = teams > 1 ? static_cast<size_t>(teams) * width * sizeof(float) : 0;
            const int grid = gridFor(reinterpret_cast<const void *>(kernel), (rows + kGradRowsOfTeam - 1) / kGradRowsOfTeam, teams, plan.threads, smem);
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
            NormGradient p{rows, width, plan.warps, dy_dev, dtotal_dev, x_dev, residual_dev, weight_dev, x_pitch, residual_pitch, rms_dev, weight_type, dx_dev, nullptr};
            if (dweight_dev) p.partial = Workspace(workspace_dev, workspace_bytes).take<float>(static_cast<size_t>(grid) * width);
            if (!dweight_dev) smem = 0;
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
