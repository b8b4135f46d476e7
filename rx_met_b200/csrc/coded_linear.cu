// Product of 8-bit codes with an epilogue.  Entry point, and the kernel for operands whose rows do not start on 16 bytes.
#include "coded_linear.cuh"
#include "dependent_launch.cuh"

namespace rxmet {
namespace codedlinear {

constexpr int kTile = 64;

namespace {

// A CTA computes 64 rows x 64 channels; 64 codes of K at a time go to shared memory byte by byte, packed in words of four for dp4a.
constexpr int kWords = 16, kThreads = 256;

__device__ __forceinline__ uint32_t wordAt(const int8_t *row, int k, int inner) {
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (k + i < inner) word |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * i);
    return word;
}

template <class T>
__global__ void __launch_bounds__(kThreads) codedLinearBytes(const __grid_constant__ Problem p) {
    __shared__ uint32_t a[kWords][kTile + 1], b[kWords][kTile + 1];
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kTile;
    const int col0 = blockIdx.x * kTile;
    waitForPredecessor();
    letDependentsStart();
    int32_t acc[4][4] = {};
    for (int k0 = 0; k0 < p.inner; k0 += kWords * 4) {
        for (int i = tid; i < kTile * kWords; i += kThreads) {
            const int r = i / kWords, w = i % kWords, k = k0 + 4 * w;
            a[w][r] = row0 + r < p.rows ? wordAt(p.codes + (row0 + r) * p.codesPitch, k, p.inner) : 0u;
            b[w][r] = col0 + r < p.outer ? wordAt(p.weight + static_cast<int64_t>(col0 + r) * p.weightPitch, k, p.inner) : 0u;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            int av[4], bv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                av[i] = static_cast<int>(a[w][ty + 16 * i]);
                bv[i] = static_cast<int>(b[w][tx + 16 * i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = col0 + tx + 16 * j;
        if (n >= p.outer) continue;
        const Channel channel(p, n);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = channel.value(acc[i][j], p.scale[min(row0 + ty + 16 * i, p.rows - 1)]);
        activate(v, p.activation);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = row0 + ty + 16 * i;
            if (m >= p.rows) continue;
            if (p.residual) v[i] += toFloat(static_cast<const T *>(p.residual)[m * p.residualPitch + n]);
            static_cast<T *>(p.out)[m * p.outer + n] = fromFloat<T>(v[i]);
        }
    }
}

void launchBytes(const Problem &p, cudaStream_t st) {
    const dim3 grid((p.outer + kTile - 1) / kTile, static_cast<unsigned>((p.rows + kTile - 1) / kTile));
    withType(p.outType, [&](auto t) {
        {
            KernelTimer timer__("codedLinearBytes", st);
            launchDependent(codedLinearBytes<decltype(t)>, grid, kThreads, 0, st, p);
        }
        afterLaunch("codedLinearBytes");
    });
}

}  // namespace
}  // namespace codedlinear
}  // namespace rxmet

using namespace rxmet;

extern "C" int rxmet_coded_linear(int64_t rows, int inner, int outer, const int8_t *codes_dev, int64_t codes_pitch, const float *scale_dev,
                                  const int8_t *weight_dev, int64_t weight_pitch, const float *weight_scale_dev, const float *bias_dev,
                                  int activation, const void *residual_dev, int64_t residual_pitch, int out_type, void *out_dev, void *stream) {
    return guarded([&] {
        RXMET_REQUIRE(rows >= 0 && inner >= 1 && outer >= 1, "coded_linear: %lld rows, inner %d, outer %d", static_cast<long long>(rows), inner, outer);
        // -128 * -128 * inner has to stay below 2^31
        if (inner > 131071) fail(RXMET_ERR_UNSUPPORTED, "coded_linear: inner %d, at most 131071", inner);
        // tiles of 64 along a grid axis of 65535
        constexpr int64_t kMost = int64_t{65535} * codedlinear::kTile;
        if (rows > kMost || outer > kMost) fail(RXMET_ERR_UNSUPPORTED, "coded_linear: %lld rows, outer %d, at most %lld each", static_cast<long long>(rows), outer, static_cast<long long>(kMost));
        RXMET_REQUIRE(activation >= RXMET_ACTIVATION_NONE && activation <= RXMET_ACTIVATION_GELU, "coded_linear: unknown activation %d", activation);
        if (rows == 0) return;
        RXMET_REQUIRE(codes_dev && scale_dev && weight_dev && weight_scale_dev && out_dev, "coded_linear: null tensor");
        RXMET_REQUIRE((rows == 1 || codes_pitch >= inner) && (outer == 1 || weight_pitch >= inner), "coded_linear: rows overlap");
        if (rows == 1) codes_pitch = static_cast<int64_t>(alignUp(inner, 16));   // the distance of a single row's next one does not matter
        if (outer == 1) weight_pitch = static_cast<int64_t>(alignUp(inner, 16));
        const codedlinear::Problem p{rows, inner, outer, codes_dev, codes_pitch, scale_dev, weight_dev, weight_pitch, weight_scale_dev, bias_dev, activation,
                                     residual_dev, residual_pitch, out_type, out_dev};
        if (codedlinear::takesTensorCores(p)) codedlinear::launchTensorCores(p, static_cast<cudaStream_t>(stream));
        else codedlinear::launchBytes(p, static_cast<cudaStream_t>(stream));
    });
}
