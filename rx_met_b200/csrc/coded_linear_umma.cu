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

// What the epilogue of sixteen rows reads from memory, asked for before the rows in front of them are worked on: lane j holds the scale of row j % N.
template <class T, int N = 16>
struct RowInputs {
    float scale;
    T residual[N];
    __device__ __forceinline__ void load(const Problem &p, int n, int64_t row0, int count) {
        const int j = threadIdx.x & (N - 1);
        scale = j < count ? p.scale[row0 + j] : 0.f;
        if (p.residual && n < p.outer) {
            const T *from = static_cast<const T *>(p.residual) + row0 * p.residualPitch + n;
#pragma unroll
            for (int i = 0; i < N; ++i, from += p.residualPitch)
                if (i < count) residual[i] = *from;
        }
    }
};
// N rows of the accumulator, one channel: epilogue and stores of those below `count`.  All lanes of a warp take part.
template <class T, int N>
__device__ __forceinline__ void storeRows(const Problem &p, const Channel &channel, int n, int64_t row0, int count, const RowInputs<T, N> &in, const uint32_t (&acc)[N]) {
    float y[N];
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = channel.value(static_cast<int32_t>(acc[j]), __shfl_sync(0xffffffffu, in.scale, j));
    activate(y, p.activation);
    if (p.residual) {
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] += toFloat(in.residual[j]);
    }
    if (n >= p.outer) return;
    T *to = static_cast<T *>(p.out) + row0 * p.outer + n;
#pragma unroll
    for (int j = 0; j < N; ++j, to += p.outer)
        if (j < count) *to = fromFloat<T>(y[j]);
}

// ---- many rows ----------------------------------------------------------------------------------------------------------

constexpr int kPairRows = 256, kPairStages = 6, kPairEpilogueWarps = 16;
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
        constexpr int kGroupRows = kPairRows / (kPairEpilogueWarps / 4);   // rows of a tile that a group of four warps takes, kPart at a time
        constexpr int kPart = 8;
        const int quarter = warp & 3, group = warp >> 2;
        int item = 0;
        for (int tile = blockIdx.x / 2; tile < tiles; tile += pairs, ++item) {
            int channelTile, rowTile;
            place(tile, channelTile, rowTile);
            const uint32_t buf = item & 1;
            const int n = channelTile * 2 * kChannels + rank * kChannels + 32 * quarter + lane;
            const Channel channel(p, min(n, p.outer - 1));
            const int64_t first = static_cast<int64_t>(rowTile) * kPairRows + group * kGroupRows;
            const int count = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(kGroupRows), p.rows - first)));
            RowInputs<T, kPart> in;
            in.load(p, n, first, count);
            wait(&accFull[buf], (item >> 1) & 1);
            fenceAfter();
            const uint32_t from = tmem + (static_cast<uint32_t>(32 * quarter) << 16) + buf * kPairRows + group * kGroupRows;
#pragma unroll 1
            for (int at = 0; at < kGroupRows; at += kPart) {
                uint32_t acc[kPart];
                const RowInputs<T, kPart> now = in;
                in.load(p, n, first + at + kPart, count - at - kPart);
                loadTmem8(from + at, acc);
                loadsDone();
                if (at + kPart == kGroupRows) {
                    fenceBefore();
                    __syncwarp();
                    if (lane == 0) arriveRemote(cluster::remote(smemAddr(&accFree[buf]), 0));
                }
                if (alive) storeRows<T>(p, channel, n, first + at, count - at, now, acc);
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
    static constexpr int kStages = NR <= 32 ? 9 : NR == 64 ? 8 : 6;   // 160 to 192 KB in flight, one CTA an SM
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
            RowInputs<T> in;
            in.load(p, n, row0, count);
#pragma unroll 1
            for (int col = 0; col < count; col += 16) {
                uint32_t acc[16];
                const RowInputs<T> now = in;
                in.load(p, n, row0 + col + 16, count - col - 16);
                loadTmem16(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + col, acc);
                loadsDone();
                if (alive) storeRows<T>(p, channel, n, row0 + col, count - col, now, acc);
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
        // the CTA adds up every `parts`th group of eight rows of all CTAs
        if (warp >= 2) {
            const Channel channel(p, min(n, p.outer - 1));
            for (int first = 8 * part; first < count; first += 8 * parts) {
                RowInputs<T, 8> in;
                in.load(p, n, row0 + first, count - first);
                uint32_t sum[8] = {};
                for (int from = 0; from < parts; ++from) {
                    const uint32_t at = cluster::remote(stages, from) + (first * kChannels + 32 * quarter + lane) * 4;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t v;
                        asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(at + j * kChannels * 4) : "memory");
                        sum[j] += v;
                    }
                }
                if (complete) storeRows<T>(p, channel, n, row0 + first, count - first, in, sum);
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
size_t splitShared() {
    return std::max<size_t>(Split<NR>::kBytes, cluster::leastShared(Split<NR>::kTmemCols));
}
// CTAs of clusters of `parts` that the device holds at the same time, asked once a process (its GPUs are alike).
template <int NR>
int residentParts(int parts) {
    if (parts == 1) return currentDevice().sms;
    static std::atomic<int> known[9];
    if (const int n = known[parts].load(std::memory_order_relaxed)) return n;
    const void *kernel = reinterpret_cast<const void *>(codedLinearSplit<float, NR>);
    ensureDynamicSmem(kernel, splitShared<NR>());
    const int n = std::max(1, residentClusters(kernel, parts, kSplitThreads, splitShared<NR>())) * parts;
    known[parts].store(n, std::memory_order_relaxed);
    return n;
}

template <int NR>
void launchSplit(const Problem &p, int parts, cudaStream_t st) {
    const CUtensorMap weights = rowsMap(p.weight, p.outer, p.inner, p.weightPitch, kChannels), codes = rowsMap(p.codes, p.rows, p.inner, p.codesPitch, NR);
    withType(p.outType, [&](auto t) {
        const auto kernel = codedLinearSplit<decltype(t), NR>;
        const size_t smem = splitShared<NR>();
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

// Which kernel, row tile and number of parts: the least of these estimates, fitted to 700 measured calls of 1 to 2048 rows, K 512 to 4096, 1024 to 8192 channels.  In
// microseconds: a chunk of K takes a cluster's CTA 0.24 whatever its rows and a pair 0.28; a CTA of few rows begins and ends in 2.8 to 5.8, a sum over parts adds 1.6 to
// 2.9, and a pair's epilogue takes 3, under the next tile's products if there is one.  K = N = 4096: 16 rows 6.2 in four parts (10.5 in one, pairs 16), 128 rows 9.5
// (pairs 16), 512 rows 14.9 (64-row tiles 24), 1024 rows 17.9 in pairs (29 in 128-row tiles).
void launchTensorCores(const Problem &p, cudaStream_t st) {
    bindContext();
    const int sms = currentDevice().sms, chunks = (p.inner + kChunk - 1) / kChunk;
    auto over = [](int64_t a, int64_t b) { return static_cast<double>((a + b - 1) / b); };
    const double pairTile = 0.28 * chunks, pairEnd = 3.0;
    double best = 3.0 + over(static_cast<int64_t>(over(p.outer, 2 * kChannels)) * static_cast<int64_t>(over(p.rows, kPairRows)), sms / 2) * std::max(pairTile, pairEnd) +
                  std::min(pairTile, pairEnd);
    int rows = 0, parts = 1;
    for (const int r : {16, 32, 64, 128})
        for (int q = 1; q <= 8 && q <= chunks; q *= 2) {
            if (p.rows > int64_t{65535} * r) continue;   // of a grid's axis
            const int64_t ctas = static_cast<int64_t>(over(p.outer, kChannels)) * static_cast<int64_t>(over(p.rows, r)) * q;
            const int resident = r == 16 ? residentParts<16>(q) : r == 32 ? residentParts<32>(q) : r == 64 ? residentParts<64>(q) : residentParts<128>(q);
            const double ends = r == 16 ? 2.8 : r == 32 ? 3.3 : r == 64 ? 4.5 : 5.8;
            const double time = over(ctas, resident) * (ends + 0.24 * over(chunks, q)) + (q > 1 ? 1.3 + 0.1 * q + 0.8 * r / 128 : 0.0);
            if (time < best) {
                best = time;
                rows = r;
                parts = q;
            }
        }
    if (rows == 0) launchPairs(p, st);
    else if (rows == 16) launchSplit<16>(p, parts, st);
    else if (rows == 32) launchSplit<32>(p, parts, st);
    else if (rows == 64) launchSplit<64>(p, parts, st);
    else launchSplit<128>(p, parts, st);
}

}  // namespace codedlinear
}  // namespace rxmet

extern "C" int rxmet_wait_status(int *gave_up) {
    return rxmet::guarded([&] {
        RXMET_REQUIRE(gave_up, "wait_status: null pointer");
        RXMET_CUDA(cudaDeviceSynchronize());   // the copy alone waits for the legacy stream, and not for streams apart from it
        RXMET_CUDA(cudaMemcpy(gave_up, rxmet::waitStatus(), sizeof(int), cudaMemcpyDeviceToHost));
    });
}
