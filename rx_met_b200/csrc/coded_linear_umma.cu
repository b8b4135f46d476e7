// Product of 8-bit codes with an epilogue on tcgen05 kind::i8, exact 32-bit integer sums in tensor memory.
//
// Computed transposed, D[channel][row]: a lane of tensor memory is an output channel, whose scale and bias live in registers, and for one row the lanes
// of a warp load and store neighbouring channels.  Both operands come as TMA boxes of 128 codes along K; what lies beyond an array reads as zeros and adds nothing.
//
// codedLinearPairs: many rows.  A pair of CTAs computes tiles of 256 channels x 256 rows, each CTA holding half of both operands; pairs walk over tiles, and two
//   accumulators let the epilogue of a tile run under the products of the next.
// codedLinearSplit: few rows.  A tile is 128 channels x 16 to 128 rows; a cluster of CTAs shares the sum over K, because few tiles alone would leave most SMs without
//   weights to fetch.  The CTAs' parts are integers, so their sum does not depend on its order.
#include "coded_linear.cuh"
#include "dependent_launch.cuh"
#include "umma_tiles.cuh"

namespace rxmet {

namespace {
__device__ int waitGaveUp;
}
int *waitStatus() {
    static std::atomic<int *> known[64];
    const int device = currentDevice().device;
    if (int *at = device < 64 ? known[device].load() : nullptr) return at;
    void *at = nullptr;
    RXMET_CUDA(cudaGetSymbolAddress(&at, waitGaveUp));
    if (device < 64) known[device] = static_cast<int *>(at);
    return static_cast<int *>(at);
}

namespace codedlinear {
namespace {

using namespace ummatiles;

constexpr int kChunk = 128;                  // codes of K in a stage
constexpr int kChannels = 128;               // channels of a CTA's accumulator
constexpr uint32_t kWeightBytes = kChannels * kChunk;

// Sixteen rows of the accumulator, one channel: epilogue and stores of those below `count`.
template <class T, class Sums>
__device__ __forceinline__ void storeRows(const Problem &p, const Channel &channel, int n, int64_t row0, int count, Sums sums) {
    float v[16];
    if (p.residual) {
        const T *from = static_cast<const T *>(p.residual) + row0 * p.residualPitch + n;
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = j < count ? toFloat(from[j * p.residualPitch]) : 0.f;
    }
    T *to = static_cast<T *>(p.out) + row0 * p.outer + n;
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (j < count) {
            const float y = channel.value(sums(j), p.scale[row0 + j], p.activation);
            to[static_cast<int64_t>(j) * p.outer] = fromFloat<T>(p.residual ? y + v[j] : y);
        }
}

// ---- many rows ----------------------------------------------------------------------------------------------------------

constexpr int kPairRows = 256, kPairStages = 6, kPairEpilogueWarps = 8;
constexpr int kPairThreads = 32 * (kPairEpilogueWarps + 2);
constexpr uint32_t kPairStageBytes = 2 * kWeightBytes;   // a CTA's 128 channels and its 128 rows
constexpr uint32_t kPairShared = 231936;                 // cluster::leastShared(512)

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    codedLinearPairs(const __grid_constant__ Problem p, const __grid_constant__ CUtensorMap weightMap, const __grid_constant__ CUtensorMap codeMap, int *status) {
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t full[kPairStages], freed[kPairStages], accFull[2], accFree[2];
    __shared__ uint32_t tmemSlot;
    const uint32_t stages = (smemAddr(raw) + 1023u) & ~1023u;
    const int warp = warpIndex(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster::rank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kPairStages; ++i) { cluster::initBarrier(&full[i], 1); cluster::initBarrier(&freed[i], 1); }
        for (int i = 0; i < 2; ++i) { cluster::initBarrier(&accFull[i], 1); cluster::initBarrier(&accFree[i], 2 * kPairEpilogueWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetchMap(&weightMap);
        prefetchMap(&codeMap);
    }
    if (warp == 0) allocTmem<2>(smemAddr(&tmemSlot), 512);
    fenceBefore();
    __syncthreads();
    cluster::barrierAll();
    fenceAfter();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmemSlot, 0);
    waitForPredecessor();
    letDependentsStart();

    const int chunks = (p.inner + kChunk - 1) / kChunk;
    const int channelTiles = (p.outer + 2 * kChannels - 1) / (2 * kChannels), rowTiles = static_cast<int>((p.rows + kPairRows - 1) / kPairRows);
    const int tiles = channelTiles * rowTiles, pairs = gridDim.x / 2;
    // Tiles in columns of eight row tiles, so that the pairs at work at the same time share rows as well as channels.
    auto place = [&](int tile, int &channelTile, int &rowTile) {
        const int group = tile / (8 * channelTiles), first = group * 8, rows = min(8, rowTiles - first), in = tile - group * 8 * channelTiles;
        channelTile = in / rows;
        rowTile = first + in - channelTile * rows;
    };
    bool alive = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (alive) alive = __all_sync(0xffffffffu, waitSuspended(smemAddr(bar), parity));
    };

    if (warp == kPairEpilogueWarps) {   // copies
        Turn turn;
        for (int tile = blockIdx.x / 2; tile < tiles; tile += pairs) {
            int channelTile, rowTile;
            place(tile, channelTile, rowTile);
            for (int c = 0; c < chunks; ++c, turn.step(kPairStages)) {
                if (turn.again) wait(&freed[turn.at], turn.parity ^ 1u);
                if (alive && electOne()) {
                    const uint32_t bar = smemAddr(&full[turn.at]), to = stages + turn.at * kPairStageBytes;
                    if (rank == 0) cluster::arriveExpect(bar, 2 * kPairStageBytes);
                    copyTile2Pair(to, &weightMap, c * kChunk, channelTile * 2 * kChannels + rank * kChannels, bar);
                    copyTile2Pair(to + kWeightBytes, &codeMap, c * kChunk, rowTile * kPairRows + rank * (kPairRows / 2), bar);
                }
                __syncwarp();
            }
        }
        // nothing is left in flight: the last use of each stage is read before this CTA ends
        for (int i = 0; i < kPairStages; ++i, turn.step(kPairStages))
            if (turn.again) waitSuspended(smemAddr(&freed[turn.at]), turn.parity ^ 1u);
    } else if (warp == kPairEpilogueWarps + 1) {   // products, issued by the first CTA for both
        if (rank == 0) {
            Turn turn;
            int item = 0;
            constexpr uint32_t kIdesc = signedCodes(2 * kChannels, kPairRows);
            for (int tile = blockIdx.x / 2; tile < tiles; tile += pairs, ++item) {
                const uint32_t buf = item & 1;
                if (item > 1) wait(&accFree[buf], ((item >> 1) - 1) & 1);
                fenceAfter();
                for (int c = 0; c < chunks; ++c, turn.step(kPairStages)) {
                    wait(&full[turn.at], turn.parity);
                    if (alive && electOne()) {
                        fenceAfter();
                        const uint32_t at = stages + turn.at * kPairStageBytes;
                        const uint64_t a = swizzledDescriptor(at), b = swizzledDescriptor(at + kWeightBytes);
#pragma unroll
                        for (int k = 0; k < kChunk / 32; ++k) productI8<2>(tmem + buf * kPairRows, a + 2 * k, b + 2 * k, kIdesc, c + k > 0 ? 1u : 0u);
                        commitPair(smemAddr(&freed[turn.at]));
                        if (c + 1 == chunks) commitPair(smemAddr(&accFull[buf]));
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        int item = 0;
        for (int tile = blockIdx.x / 2; tile < tiles; tile += pairs, ++item) {
            int channelTile, rowTile;
            place(tile, channelTile, rowTile);
            const uint32_t buf = item & 1;
            const int n = channelTile * 2 * kChannels + rank * kChannels + 32 * quarter + lane;
            const Channel channel(p, min(n, p.outer - 1));
            wait(&accFull[buf], (item >> 1) & 1);
            fenceAfter();
#pragma unroll 1
            for (int part = 0; part < kPairRows / 32; ++part) {
                uint32_t acc[16];
                const int col = half * (kPairRows / 2) + part * 16;
                loadTmem16(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + buf * kPairRows + col, acc);
                loadsDone();
                if (part + 1 == kPairRows / 32) {
                    fenceBefore();
                    __syncwarp();
                    if (lane == 0) arriveRemote(cluster::remote(smemAddr(&accFree[buf]), 0));
                }
                const int64_t row0 = static_cast<int64_t>(rowTile) * kPairRows + col;
                if (alive && n < p.outer) storeRows<T>(p, channel, n, row0, static_cast<int>(min(static_cast<int64_t>(16), p.rows - row0)), [&](int j) { return static_cast<int32_t>(acc[j]); });
            }
        }
    }
    if (!alive && lane == 0) atomicExch(status, 1);
    fenceBefore();
    __syncthreads();
    cluster::barrierAll();
    if (warp == 0) freeTmem<2>(tmem, 512);
}

// ---- few rows -----------------------------------------------------------------------------------------------------------

constexpr int kSplitThreads = 192;

template <int NR>
struct Split {
    static constexpr uint32_t kStageBytes = kWeightBytes + NR * kChunk;
    static constexpr int kStages = NR <= 32 ? 5 : NR == 64 ? 4 : 3;   // two CTAs an SM
    static constexpr uint32_t kTmemCols = NR < 32 ? 32 : NR;
    static constexpr uint32_t kBytes = kStages * kStageBytes + 1024;   // the parts of the sums, NR x 128 integers, fit the stages
};

// blockIdx: x = part of the sum over K (the cluster), y = channel tile, z = row tile.
template <class T, int NR>
__global__ void __launch_bounds__(kSplitThreads) codedLinearSplit(const __grid_constant__ Problem p, const __grid_constant__ CUtensorMap weightMap,
                                                                  const __grid_constant__ CUtensorMap codeMap, int *status) {
    using S = Split<NR>;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t full[S::kStages], freed[S::kStages], accFull;
    __shared__ uint32_t tmemSlot;
    __shared__ int failed;
    const uint32_t stages = (smemAddr(raw) + 1023u) & ~1023u;
    const int warp = warpIndex(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        failed = 0;
        for (int i = 0; i < S::kStages; ++i) { cluster::initBarrier(&full[i], 1); cluster::initBarrier(&freed[i], 1); }
        cluster::initBarrier(&accFull, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetchMap(&weightMap);
        prefetchMap(&codeMap);
    }
    if (warp == 1) allocTmem<1>(smemAddr(&tmemSlot), S::kTmemCols);
    fenceBefore();
    __syncthreads();
    fenceAfter();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmemSlot, 0);
    waitForPredecessor();
    letDependentsStart();

    const int all = (p.inner + kChunk - 1) / kChunk, parts = gridDim.x, part = blockIdx.x;
    const int firstChunk = static_cast<int>(static_cast<int64_t>(all) * part / parts), chunks = static_cast<int>(static_cast<int64_t>(all) * (part + 1) / parts) - firstChunk;
    const int n0 = blockIdx.y * kChannels;
    const int64_t row0 = static_cast<int64_t>(blockIdx.z) * NR;
    bool alive = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (alive) alive = __all_sync(0xffffffffu, waitSuspended(smemAddr(bar), parity));
    };
    if (warp == 0) {
        Turn turn;
        for (int c = 0; c < chunks; ++c, turn.step(S::kStages)) {
            if (turn.again) wait(&freed[turn.at], turn.parity ^ 1u);
            if (alive && electOne()) {
                const uint32_t bar = smemAddr(&full[turn.at]), to = stages + turn.at * S::kStageBytes;
                cluster::arriveExpect(bar, S::kStageBytes);
                copyTile2(to, &weightMap, (firstChunk + c) * kChunk, n0, bar);
                copyTile2(to + kWeightBytes, &codeMap, (firstChunk + c) * kChunk, static_cast<int>(row0), bar);
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        Turn turn;
        constexpr uint32_t kIdesc = signedCodes(kChannels, NR);
        for (int c = 0; c < chunks; ++c, turn.step(S::kStages)) {
            wait(&full[turn.at], turn.parity);
            if (alive && electOne()) {
                fenceAfter();
                const uint32_t at = stages + turn.at * S::kStageBytes;
                const uint64_t a = swizzledDescriptor(at), b = swizzledDescriptor(at + kWeightBytes);
#pragma unroll
                for (int k = 0; k < kChunk / 32; ++k) productI8<1>(tmem, a + 2 * k, b + 2 * k, kIdesc, c + k > 0 ? 1u : 0u);
                commitTo(smemAddr(&freed[turn.at]));
                if (c + 1 == chunks) commitTo(smemAddr(&accFull));
            }
            __syncwarp();
        }
    }
    // every CTA has a chunk, so that its accumulator is written; then all copies have landed and all stages are read
    wait(&accFull, 0);
    fenceAfter();
    const int quarter = warp & 3, count = static_cast<int>(min(static_cast<int64_t>(NR), p.rows - row0));
    const int n = n0 + 32 * quarter + lane;
    if (warp >= 2) {
        if (parts == 1) {
            const Channel channel(p, min(n, p.outer - 1));
#pragma unroll 1
            for (int col = 0; col < NR; col += 16) {
                uint32_t acc[16];
                loadTmem16(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + col, acc);
                loadsDone();
                if (alive && n < p.outer && col < count) storeRows<T>(p, channel, n, row0 + col, min(16, count - col), [&](int j) { return static_cast<int32_t>(acc[j]); });
            }
        } else {
#pragma unroll 1
            for (int col = 0; col < count; col += 16) {
                uint32_t acc[16];
                loadTmem16(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + col, acc);
                loadsDone();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(stages + ((col + j) * kChannels + 32 * quarter + lane) * 4), "r"(acc[j]) : "memory");
            }
        }
    }
    if (!alive) failed = 1;
    if (parts > 1) {
        __syncthreads();
        const bool complete = failed == 0;
        cluster::barrierAll();
        // the CTA adds up every `parts`th group of four rows of all CTAs
        if (warp >= 2 && n < p.outer) {
            const Channel channel(p, n);
            for (int first = 4 * part; first < count; first += 4 * parts) {
                int32_t sum[4] = {};
                for (int from = 0; from < parts; ++from) {
                    const uint32_t at = cluster::remote(stages, from);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        int32_t v;
                        asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(at + ((first + j) * kChannels + 32 * quarter + lane) * 4) : "memory");
                        sum[j] += v;
                    }
                }
                if (complete) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (first + j < count) {
                            const int64_t m = row0 + first + j;
                            float y = channel.value(sum[j], p.scale[m], p.activation);
                            if (p.residual) y += toFloat(static_cast<const T *>(p.residual)[m * p.residualPitch + n]);
                            static_cast<T *>(p.out)[m * p.outer + n] = fromFloat<T>(y);
                        }
                }
            }
        }
        __syncwarp();
        cluster::barrierAll();
    }
    fenceBefore();
    __syncthreads();
    if (failed && threadIdx.x == 0) atomicExch(status, 1);
    if (warp == 1) freeTmem<1>(tmem, S::kTmemCols);
}

CUtensorMap rowsMap(const int8_t *data, int64_t rows, int inner, int64_t pitch, int boxRows) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(pitch)};
    const cuuint32_t box[2] = {kChunk, static_cast<cuuint32_t>(boxRows)}, steps[2] = {1, 1};
    const CUresult rc = encodeTiled()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(data), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) fail(RXMET_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", static_cast<int>(rc));
    return map;
}

template <int NR>
void launchSplit(const Problem &p, int parts, cudaStream_t st) {
    using S = Split<NR>;
    const CUtensorMap weights = rowsMap(p.weight, p.outer, p.inner, p.weightPitch, kChannels), codes = rowsMap(p.codes, p.rows, p.inner, p.codesPitch, NR);
    withType(p.outType, [&](auto t) {
        const auto kernel = codedLinearSplit<decltype(t), NR>;
        const size_t smem = std::max<size_t>(S::kBytes, cluster::leastShared(S::kTmemCols));
        ensureDynamicSmem(reinterpret_cast<const void *>(kernel), smem);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(parts, (p.outer + kChannels - 1) / kChannels, static_cast<unsigned>((p.rows + NR - 1) / NR));
        cfg.blockDim = kSplitThreads;
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attrs[2] = {};
        attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[0].val.programmaticStreamSerializationAllowed = 1;
        attrs[1].id = cudaLaunchAttributeClusterDimension;
        attrs[1].val.clusterDim.x = parts;
        attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
        cfg.attrs = attrs;
        cfg.numAttrs = 2;
        {
            KernelTimer timer__("codedLinearSplit", st);
            RXMET_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, weights, codes, waitStatus()));
        }
        afterLaunch("codedLinearSplit");
    });
}

void launchPairs(const Problem &p, cudaStream_t st) {
    const CUtensorMap weights = rowsMap(p.weight, p.outer, p.inner, p.weightPitch, kChannels), codes = rowsMap(p.codes, p.rows, p.inner, p.codesPitch, kPairRows / 2);
    withType(p.outType, [&](auto t) {
        const auto kernel = codedLinearPairs<decltype(t)>;
        ensureDynamicSmem(reinterpret_cast<const void *>(kernel), kPairShared);
        const int64_t tiles = static_cast<int64_t>((p.outer + 2 * kChannels - 1) / (2 * kChannels)) * ((p.rows + kPairRows - 1) / kPairRows);
        const int grid = 2 * static_cast<int>(std::min<int64_t>(currentDevice().sms / 2, tiles));
        {
            KernelTimer timer__("codedLinearPairs", st);
            launchDependent(kernel, grid, kPairThreads, kPairShared, st, p, weights, codes, waitStatus());
        }
        afterLaunch("codedLinearPairs");
    });
}

}  // namespace

bool takesTensorCores(const Problem &p) {
    return encodeTiled() != nullptr && p.codesPitch % 16 == 0 && p.weightPitch % 16 == 0 && alignedTo(p.codes, 16) && alignedTo(p.weight, 16);
}

void launchTensorCores(const Problem &p, cudaStream_t st) {
    const int sms = currentDevice().sms, chunks = (p.inner + kChunk - 1) / kChunk, channelTiles = (p.outer + kChannels - 1) / kChannels;
    if (p.rows > 512) return launchPairs(p, st);
    const int rows = p.rows <= 16 ? 16 : p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : 128;
    const int64_t tiles = static_cast<int64_t>(channelTiles) * ((p.rows + rows - 1) / rows);
    int parts = 1;
    while (parts < 8 && tiles * parts * 2 <= 2 * sms && parts * 2 <= chunks) parts *= 2;
    if (rows == 16) launchSplit<16>(p, parts, st);
    else if (rows == 32) launchSplit<32>(p, parts, st);
    else if (rows == 64) launchSplit<64>(p, parts, st);
    else launchSplit<128>(p, parts, st);
}

}  // namespace codedlinear
}  // namespace rxmet

extern "C" int rxmet_wait_status(int *gave_up) {
    return rxmet::guarded([&] {
        RXMET_REQUIRE(gave_up, "wait_status: null pointer");
        RXMET_CUDA(cudaMemcpy(gave_up, rxmet::waitStatus(), sizeof(int), cudaMemcpyDeviceToHost));
    });
}
