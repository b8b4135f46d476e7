// Gated linear recurrence: entry points, the forward pass over sequences, and single tokens.
//
// Forward: a tile's gates are worked out once and stay in registers, (f, z c) of sixteen tokens a thread; the state in front of the tile comes from the chain, and a second walk over the
// registers gives the outputs.  So every input is read once and every output written once, whatever the length.
#include "gated_recurrence.cuh"

namespace rxmet {
namespace gated {
namespace {

constexpr int kStages = 2;

template <class T, int PIECE, bool OWN>
__global__ void __launch_bounds__(kThreads, 2) gatedForward(const __grid_constant__ Pass p) {
    constexpr int N = kLane<T>, kTensors = OWN ? 3 : 2;
    extern __shared__ __align__(128) uint8_t stages[];
    __shared__ float2 window[kWindow][32 * N], parts[kWarps][32 * N];
    __shared__ int64_t tileOf[kStages];
    __shared__ int nearest;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    waitForPredecessor();
    letDependentsStart();
    Tickets tickets(p);
    if (tid == 0)
        for (int i = 0; i < kStages; ++i) tileOf[i] = tickets.take();
    __syncthreads();
    auto ask = [&](int stage) {
        const int64_t index = tileOf[stage];
        if (index < p.tiles) {
            const Tile<T> tile(p, index, false);
            const uint32_t to = umma::smemAddr(stages) + stage * kTensors * kTensorBytes<T>;
            askFor<T, PIECE>(to, p.forget, tile, p.width);
            askFor<T, PIECE>(to + kTensorBytes<T>, p.value, tile, p.width);
            if (OWN) askFor<T, PIECE>(to + 2 * kTensorBytes<T>, p.input, tile, p.width);
        }
        commitCopies();
    };
    for (int i = 0; i < kStages; ++i) ask(i);

    for (int stage = 0;; stage = (stage + 1) % kStages) {
        const int64_t index = tileOf[stage];
        if (index >= p.tiles) break;
        const Tile<T> tile(p, index, false);
        int64_t later = 0;
        if (tid == 0) later = tickets.take();
        copiesArrived<kStages - 1>();
        __syncthreads();

        const uint8_t *from = stages + stage * kTensors * kTensorBytes<T> + (warp * kSteps * 32 + lane) * N * sizeof(T);
        const int live = tile.live - warp * kSteps;   // of this warp's tokens
        float a[kSteps][N], b[kSteps][N], A[N], B[N];
#pragma unroll
        for (int v = 0; v < N; ++v) {
            A[v] = 1.f;
            B[v] = 0.f;
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float forget[N], value[N], input[N];
            const uint8_t *row = from + s * 32 * N * sizeof(T);
            readRow<T>(row, forget);
            readRow<T>(row + kTensorBytes<T>, value);
            if (OWN) readRow<T>(row + 2 * kTensorBytes<T>, input);
#pragma unroll
            for (int v = 0; v < N; ++v) {
                const Gate f(forget[v]);
                float c = value[v], z = f.shut;
                if (p.tanhValue) c = tanhf(c);
                if (OWN) z = Gate(input[v]).open;
                a[s][v] = s < live ? f.open : 1.f;
                b[s][v] = s < live ? z * c : 0.f;
                A[v] *= a[s][v];
                B[v] = fmaf(a[s][v], B[v], b[s][v]);
            }
        }
#pragma unroll
        for (int v = 0; v < N; ++v) parts[warp][lane * N + v] = make_float2(A[v], B[v]);
        if (tid == 0) tileOf[stage] = later;
        __syncthreads();
        ask(stage);

        const int d = tile.d0 + lane * N, real = p.width - d;
        const int64_t link = tile.slab * p.chunks + tile.chunk;
        const bool last = tile.chunk + 1 == p.chunks;
        // the last warp speaks for the tile
        if (warp == kWarps - 1 && !last) {
#pragma unroll
            for (int v = 0; v < N; ++v) {
                A[v] = 1.f;
                B[v] = 0.f;
                for (int w = 0; w < kWarps; ++w) {
                    const float2 part = parts[w][lane * N + v];
                    A[v] *= part.x;
                    B[v] = fmaf(part.x, B[v], part.y);
                }
            }
            if (tile.chunk > 0) tellPart<N>(p.chain, link, A, B);
        }
        float h[N];
        if (tile.chunk > 0) stateBefore<N>(p.chain, tile.slab, tile.chunk, p.chunks, window, &nearest, h);
        else {
#pragma unroll
            for (int v = 0; v < N; ++v) h[v] = p.state && v < real ? p.state[static_cast<int64_t>(tile.b) * p.width + d + v] : 0.f;
        }
        if (warp == kWarps - 1 && !last) {
            float behind[N];
#pragma unroll
            for (int v = 0; v < N; ++v) behind[v] = fmaf(A[v], h[v], B[v]);
            tellWhole<N>(p.chain, link, behind);
        }
        if (warp == 0 && p.marks && tile.chunk > 0) {
#pragma unroll
            for (int v = 0; v < N; ++v)
                if (v < real) p.marks[(static_cast<int64_t>(tile.b) * (p.chunks - 1) + tile.chunk - 1) * p.width + d + v] = h[v];
        }
        for (int w = 0; w < warp; ++w)
#pragma unroll
            for (int v = 0; v < N; ++v) {
                const float2 part = parts[w][lane * N + v];
                h[v] = fmaf(part.x, h[v], part.y);
            }
        const int here = min(p.tokens - tile.first - warp * kSteps, kSteps);   // tokens that have an output
        T *to = static_cast<T *>(p.out) + (static_cast<int64_t>(tile.b) * p.tokens + tile.first + warp * kSteps) * p.width + d;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float y[N];
#pragma unroll
            for (int v = 0; v < N; ++v) {
                h[v] = fmaf(a[s][v], h[v], b[s][v]);
                y[v] = s < live ? h[v] : 0.f;
            }
            if (p.out && s < here) writeRow<T>(to, y, real, p.paired);
            to += p.width;
        }
        if (last && warp == kWarps - 1 && p.finalState) {
#pragma unroll
            for (int v = 0; v < N; ++v)
                if (v < real) p.finalState[static_cast<int64_t>(tile.b) * p.width + d + v] = h[v];
        }
    }
}

// Single tokens: a thread for two neighbouring channels of a row.
template <class T, bool OWN>
__global__ void __launch_bounds__(kThreads) gatedStep(const __grid_constant__ Pass p, const int pairsOfRow) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int b = static_cast<int>(i / pairsOfRow), d = 2 * static_cast<int>(i - static_cast<int64_t>(b) * pairsOfRow);
    waitForPredecessor();
    letDependentsStart();
    if (b >= p.batch) return;
    const bool live = !p.lengths || p.lengths[b] > 0;
    auto at = [&](const rxmet_token_tensor &t, int v) { return toFloat(static_cast<const T *>(t.data)[b * t.stride_b + d + v]); };
    const int64_t row = static_cast<int64_t>(b) * p.width + d;
    const int count = min(2, p.width - d);
    float forget[2], value[2], input[2], h[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int u = min(v, count - 1);
        forget[v] = at(p.forget, u);
        value[v] = at(p.value, u);
        if (OWN) input[v] = at(p.input, u);
        h[v] = p.state ? p.state[row + u] : 0.f;
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        if (v >= count) continue;
        const Gate f(forget[v]);
        const float c = p.tanhValue ? tanhf(value[v]) : value[v], z = OWN ? Gate(input[v]).open : f.shut;
        const float next = live ? fmaf(f.open, h[v], z * c) : h[v];
        if (p.finalState) p.finalState[row + v] = next;
        if (p.out) static_cast<T *>(p.out)[row + v] = fromFloat<T>(live ? next : 0.f);
    }
}

// Flags and ticket of a chain.
__global__ void __launch_bounds__(kThreads) gatedClear(int *words, int64_t count) {
    waitForPredecessor();
    letDependentsStart();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * kThreads) words[i] = 0;
}

Pass passOf(const rxmet_gated_recurrence &problem) {
    RXMET_REQUIRE(problem.batch >= 0 && problem.tokens >= 0 && problem.width >= 1, "gated_recurrence: batch %d, tokens %d, width %d", problem.batch, problem.tokens, problem.width);
    RXMET_REQUIRE(problem.type == RXMET_TYPE_F32 || problem.type == RXMET_TYPE_BF16 || problem.type == RXMET_TYPE_F16, "gated_recurrence: unknown element type %d", problem.type);
    if (problem.tokens > (1 << 30)) fail(RXMET_ERR_UNSUPPORTED, "gated_recurrence: %d tokens, at most %d", problem.tokens, 1 << 30);
    Pass p{};
    p.batch = problem.batch;
    p.tokens = problem.tokens;
    p.width = problem.width;
    const int channels = static_cast<int>(128 / typeBytes(problem.type));
    p.chunks = std::max(1, (problem.tokens + kChunk - 1) / kChunk);
    p.slabsOfRow = (problem.width + channels - 1) / channels;
    const int64_t slabs = static_cast<int64_t>(p.batch) * p.slabsOfRow;
    if (slabs * p.chunks > INT32_MAX) fail(RXMET_ERR_UNSUPPORTED, "gated_recurrence: %lld runs of %d tokens of %d channels, at most %d", static_cast<long long>(slabs * p.chunks), kChunk, channels, INT32_MAX);
    p.tiles = slabs * p.chunks;
    p.tanhValue = problem.tanh_value != 0;
    p.forget = problem.forget;
    p.value = problem.value;
    p.input = problem.input;
    p.lengths = problem.lengths;
    return p;
}
void requireData(const rxmet_gated_recurrence &problem, int64_t tiles) {
    RXMET_REQUIRE(tiles == 0 || problem.tokens == 0 || (problem.forget.data && problem.value.data), "gated_recurrence: null pointer");
}

// Links of a chain and their words; nothing for sequences of one tile.
int64_t chainWords(const Pass &p) { return p.chunks > 1 ? p.tiles + 1 : 0; }
template <class W>
void takeChain(W &&ws, const Pass &p, Chain *chain) {
    if (p.chunks == 1) return;
    if constexpr (std::is_same_v<std::decay_t<W>, WorkspaceSizer>) {
        ws.template take<int>(chainWords(p));
        ws.template take<float2>(p.tiles * 64);
        ws.template take<float>(p.tiles * 64);
    } else {
        int *words = ws.template take<int>(chainWords(p));
        chain->ticket = reinterpret_cast<unsigned *>(words);
        chain->flags = words + 1;
        chain->parts = ws.template take<float2>(p.tiles * 64);
        chain->whole = ws.template take<float>(p.tiles * 64);
    }
}
void startChain(Pass &p, void *workspace, size_t bytes, cudaStream_t st) {
    p.chain.status = waitStatus();
    if (p.chunks == 1) return;
    takeChain(Workspace(workspace, bytes), p, &p.chain);
    const int64_t words = chainWords(p);
    {
        KernelTimer timer__("gatedClear", st);
        launchDependent(gatedClear, static_cast<unsigned>(std::min<int64_t>((words + kThreads - 1) / kThreads, 4 * currentDevice().sms)), kThreads, 0, st,
                        reinterpret_cast<int *>(p.chain.ticket), words);
    }
    afterLaunch("gatedClear");
}

}  // namespace

void launchForward(const Pass &p, int type, cudaStream_t st) {
    const size_t size = typeBytes(type);
    int piece = std::min(pieceOf(p.forget, p.batch, p.tokens, size), pieceOf(p.value, p.batch, p.tokens, size));
    if (p.input.data) piece = std::min(piece, pieceOf(p.input, p.batch, p.tokens, size));
    withType(type, [&](auto t) {
        using T = decltype(t);
        auto launch = [&](auto own) {
            constexpr bool kOwn = decltype(own)::value;
            withPiece<T>(piece, [&](auto bytes) {
                const auto kernel = gatedForward<T, decltype(bytes)::value, kOwn>;
                const size_t smem = kStages * (kOwn ? 3 : 2) * kTensorBytes<T>;
                ensureDynamicSmem(reinterpret_cast<const void *>(kernel), smem);
                const int resident = residentPerSm(reinterpret_cast<const void *>(kernel), kThreads, smem) * currentDevice().sms;
                {
                    KernelTimer timer__("gatedForward", st);
                    launchDependent(kernel, static_cast<unsigned>(std::min<int64_t>(p.tiles, resident)), kThreads, smem, st, p);
                }
                afterLaunch("gatedForward");
            });
        };
        if (p.input.data) launch(std::true_type{});
        else launch(std::false_type{});
    });
}

namespace {
void launchStep(const Pass &p, int type, cudaStream_t st) {
    const int pairs = (p.width + 1) / 2;
    const int64_t blocks = (static_cast<int64_t>(p.batch) * pairs + kThreads - 1) / kThreads;
    withType(type, [&](auto t) {
        using T = decltype(t);
        {
            KernelTimer timer__("gatedStep", st);
            launchDependent(p.input.data ? gatedStep<T, true> : gatedStep<T, false>, static_cast<unsigned>(blocks), kThreads, 0, st, p, pairs);
        }
        afterLaunch("gatedStep");
    });
}
}  // namespace

}  // namespace gated
}  // namespace rxmet

using namespace rxmet;

extern "C" size_t rxmet_gated_recurrence_marks(const rxmet_gated_recurrence *problem) {
    size_t floats = 0;
    guarded([&] {
        RXMET_REQUIRE(problem, "gated_recurrence: null pointer");
        const gated::Pass p = gated::passOf(*problem);
        floats = static_cast<size_t>(p.batch) * (p.chunks - 1) * p.width;
    });
    return floats;
}

extern "C" size_t rxmet_gated_recurrence_workspace_bytes(const rxmet_gated_recurrence *problem) {
    WorkspaceSizer sizer;
    guarded([&] {
        RXMET_REQUIRE(problem, "gated_recurrence: null pointer");
        gated::takeChain(sizer, gated::passOf(*problem), nullptr);
    });
    return sizer.used();
}

extern "C" int rxmet_gated_recurrence_forward(const rxmet_gated_recurrence *problem, const float *state, void *out, float *final_state, float *marks, void *workspace,
                                              size_t workspace_bytes, void *stream) {
    return guarded([&] {
        RXMET_REQUIRE(problem, "gated_recurrence: null pointer");
        gated::Pass p = gated::passOf(*problem);
        gated::requireData(*problem, p.tiles);
        if (p.tiles == 0) return;
        p.state = state;
        p.out = out;
        p.finalState = final_state;
        p.marks = marks;
        p.paired = p.width % 2 == 0 && alignedTo(out, 4);
        const auto st = static_cast<cudaStream_t>(stream);
        if (p.tokens == 1) return gated::launchStep(p, problem->type, st);
        gated::startChain(p, workspace, workspace_bytes, st);
        gated::launchForward(p, problem->type, st);
    });
}

extern "C" int rxmet_gated_recurrence_backward(const rxmet_gated_recurrence *problem, const float *state, const float *marks, const rxmet_token_tensor *dout, const float *dfinal,
                                               void *dforget, void *dvalue, void *dinput, float *dstate, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        RXMET_REQUIRE(problem, "gated_recurrence: null pointer");
        gated::Pass p = gated::passOf(*problem);
        gated::requireData(*problem, p.tiles);
        if (p.tiles == 0) return;
        RXMET_REQUIRE(marks || p.chunks == 1, "gated_recurrence backward: no marks from the forward pass");
        RXMET_REQUIRE(!dinput || problem->input.data, "gated_recurrence backward: the gradient of an input gate that is not there");
        p.state = state;
        p.marks = const_cast<float *>(marks);
        if (dout) p.dout = *dout;
        p.dfinal = dfinal;
        p.dforget = dforget;
        p.dvalue = dvalue;
        p.dinput = dinput;
        p.dstate = dstate;
        p.paired = p.width % 2 == 0 && alignedTo(dforget, 4) && alignedTo(dvalue, 4) && alignedTo(dinput, 4);
        const auto st = static_cast<cudaStream_t>(stream);
        gated::startChain(p, workspace, workspace_bytes, st);
        gated::launchBackward(p, problem->type, st);
    });
}
