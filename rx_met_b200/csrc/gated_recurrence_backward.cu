// Gated linear recurrence: the gradients.
//
//   G_t = dout_t + R_{t+1},  R_t = f_t G_t   (R behind the last token: the gradient of the final state; R_1: that of the state)
//   dvalue = G z c',  dforget = G (h_{t-1} - c) f (1 - f)  (G h_{t-1} f (1 - f) beside an input gate),  dinput = G c z (1 - z)
//
// A tile reads its gates and values again and takes the state in front of it from what the forward pass marked, so that no state of a token is kept between the passes; the gradient R that
// reaches its end comes from the chain, whose first tile is a sequence's last.  In registers: a gate (the smaller of f and 1 - f, signed) and h_{t-1} of sixteen tokens a thread;
// values and gradients are read a second time from shared memory.
#include "gated_recurrence.cuh"

namespace rxmet {
namespace gated {
namespace {

constexpr int kStages = 2;

// f and 1 - f from the smaller of them, whose sign says which it is.
__device__ __forceinline__ float packGate(const Gate &g) { return g.open > g.shut ? g.shut : -g.open; }
__device__ __forceinline__ float openOf(float packed) { return signbit(packed) ? -packed : 1.f - packed; }
__device__ __forceinline__ float shutOf(float packed) { return signbit(packed) ? 1.f + packed : packed; }

template <class T, int PIECE, bool OWN>
__global__ void __launch_bounds__(kThreads, 2) gatedBackward(const __grid_constant__ Pass p) {
    constexpr int N = kLane<T>, kTensors = OWN ? 4 : 3;
    extern __shared__ __align__(128) uint8_t stages[];
    __shared__ float2 window[kWindow][32 * N], parts[kWarps][32 * N];
    __shared__ float gradients[kWarps][32 * N];
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
            const Tile<T> tile(p, index, true);
            const uint32_t to = umma::smemAddr(stages) + stage * kTensors * kTensorBytes<T>;
            askFor<T, PIECE>(to, p.forget, tile, p.width);
            askFor<T, PIECE>(to + kTensorBytes<T>, p.value, tile, p.width);
            if (p.dout.data) askFor<T, PIECE>(to + 2 * kTensorBytes<T>, p.dout, tile, p.width);
            if (OWN) askFor<T, PIECE>(to + 3 * kTensorBytes<T>, p.input, tile, p.width);
        }
        commitCopies();
    };
    ask(0);

    for (int stage = 0;; stage ^= 1) {
        const int64_t index = tileOf[stage];
        if (index >= p.tiles) break;
        const Tile<T> tile(p, index, true);
        copiesArrived<0>();
        __syncthreads();
        ask(stage ^ 1);   // what it held was read in front of the barrier
        int64_t later = 0;
        if (tid == 0) later = tickets.take();

        const int d = tile.d0 + lane * N, real = p.width - d;
        float h[N];   // in front of the tile
#pragma unroll
        for (int v = 0; v < N; ++v) {
            const float *from = tile.chunk > 0 ? p.marks + (static_cast<int64_t>(tile.b) * (p.chunks - 1) + tile.chunk - 1) * p.width : p.state ? p.state + static_cast<int64_t>(tile.b) * p.width : nullptr;
            h[v] = from && v < real ? from[d + v] : 0.f;
        }
        const uint8_t *from = stages + stage * kTensors * kTensorBytes<T> + (warp * kSteps * 32 + lane) * N * sizeof(T);
        const int live = tile.live - warp * kSteps;
        auto values = [&](int s, float (&value)[N], float (&dout)[N]) {
            const uint8_t *row = from + s * 32 * N * sizeof(T);
            readRow<T>(row + kTensorBytes<T>, value);
            if (p.dout.data) readRow<T>(row + 2 * kTensorBytes<T>, dout);
            else
#pragma unroll
                for (int v = 0; v < N; ++v) dout[v] = 0.f;
            if (p.tanhValue)
#pragma unroll
                for (int v = 0; v < N; ++v) value[v] = tanhf(value[v]);
        };
        auto inputGates = [&](int s, float (&input)[N]) { readRow<T>(from + s * 32 * N * sizeof(T) + 3 * kTensorBytes<T>, input); };

        // the tile's maps of a state forwards, (A, B), and of a gradient backwards, (A, C)
        float gate[kSteps][N], before[kSteps][N], A[N], B[N], C[N];
#pragma unroll
        for (int v = 0; v < N; ++v) {
            A[v] = 1.f;
            B[v] = C[v] = 0.f;
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float forget[N], value[N], dout[N], input[N];
            readRow<T>(from + s * 32 * N * sizeof(T), forget);
            values(s, value, dout);
            if (OWN) inputGates(s, input);
#pragma unroll
            for (int v = 0; v < N; ++v) {
                const Gate f(forget[v]);
                gate[s][v] = packGate(f);
                const float z = OWN ? Gate(input[v]).open : f.shut;
                before[s][v] = z * value[v];   // what the token adds, until the state in front of it is known
                if (s < live) {
                    A[v] *= f.open;
                    B[v] = fmaf(f.open, B[v], before[s][v]);
                    C[v] = fmaf(A[v], dout[v], C[v]);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < N; ++v) {
            parts[warp][lane * N + v] = make_float2(A[v], B[v]);
            gradients[warp][lane * N + v] = C[v];
        }
        if (tid == 0) tileOf[stage] = later;
        __syncthreads();

        const int place = p.chunks - 1 - tile.chunk;
        const int64_t link = tile.slab * p.chunks + place;
        const bool last = tile.chunk == 0;   // of the chain
        if (warp == kWarps - 1 && !last) {
#pragma unroll
            for (int v = 0; v < N; ++v) {
                A[v] = 1.f;
                C[v] = 0.f;
                for (int w = kWarps - 1; w >= 0; --w) {
                    const float a = parts[w][lane * N + v].x;
                    A[v] *= a;
                    C[v] = fmaf(a, C[v], gradients[w][lane * N + v]);
                }
            }
            if (place > 0) tellPart<N>(p.chain, link, A, C);
        }
        float R[N];
        if (place > 0) stateBefore<N>(p.chain, tile.slab, place, p.chunks, window, &nearest, R);
        else {
#pragma unroll
            for (int v = 0; v < N; ++v) R[v] = p.dfinal && v < real ? p.dfinal[static_cast<int64_t>(tile.b) * p.width + d + v] : 0.f;
        }
        if (warp == kWarps - 1 && !last) {
            float behind[N];
#pragma unroll
            for (int v = 0; v < N; ++v) behind[v] = fmaf(A[v], R[v], C[v]);
            tellWhole<N>(p.chain, link, behind);
        }
        for (int w = 0; w < warp; ++w)
#pragma unroll
            for (int v = 0; v < N; ++v) {
                const float2 part = parts[w][lane * N + v];
                h[v] = fmaf(part.x, h[v], part.y);
            }
        for (int w = kWarps - 1; w > warp; --w)
#pragma unroll
            for (int v = 0; v < N; ++v) R[v] = fmaf(parts[w][lane * N + v].x, R[v], gradients[w][lane * N + v]);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int v = 0; v < N; ++v) {
                const float next = fmaf(openOf(gate[s][v]), h[v], before[s][v]);
                before[s][v] = h[v];
                h[v] = next;   // behind the sequence's end nobody reads it
            }
        const int here = min(p.tokens - tile.first - warp * kSteps, kSteps);
        const int64_t to = (static_cast<int64_t>(tile.b) * p.tokens + tile.first + warp * kSteps) * p.width + d;
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            float value[N], dout[N], input[N], dforget[N], dvalue[N], dinput[N];
            values(s, value, dout);
            if (OWN) inputGates(s, input);
#pragma unroll
            for (int v = 0; v < N; ++v) {
                const float f = openOf(gate[s][v]), shut = shutOf(gate[s][v]), G = s < live ? dout[v] + R[v] : 0.f;
                float z = shut, held = before[s][v] - value[v];
                if (OWN) {
                    const Gate i(input[v]);
                    z = i.open;
                    held = before[s][v];
                    dinput[v] = s < live ? G * value[v] * (i.open * i.shut) : 0.f;
                }
                dforget[v] = s < live ? G * held * (f * shut) : 0.f;
                const float slope = p.tanhValue ? fmaf(-value[v], value[v], 1.f) : 1.f;
                dvalue[v] = s < live ? G * z * slope : 0.f;
                if (s < live) R[v] = f * G;
            }
            if (s < here) {
                const int64_t at = to + static_cast<int64_t>(s) * p.width;
                if (p.dforget) writeRow<T>(static_cast<T *>(p.dforget) + at, dforget, real, p.paired);
                if (p.dvalue) writeRow<T>(static_cast<T *>(p.dvalue) + at, dvalue, real, p.paired);
                if (OWN && p.dinput) writeRow<T>(static_cast<T *>(p.dinput) + at, dinput, real, p.paired);
            }
        }
        if (last && warp == 0 && p.dstate) {
#pragma unroll
            for (int v = 0; v < N; ++v)
                if (v < real) p.dstate[static_cast<int64_t>(tile.b) * p.width + d + v] = R[v];
        }
    }
}

}  // namespace

void launchBackward(const Pass &p, int type, cudaStream_t st) {
    const size_t size = typeBytes(type);
    int piece = std::min(pieceOf(p.forget, p.batch, p.tokens, size), pieceOf(p.value, p.batch, p.tokens, size));
    if (p.dout.data) piece = std::min(piece, pieceOf(p.dout, p.batch, p.tokens, size));
    if (p.input.data) piece = std::min(piece, pieceOf(p.input, p.batch, p.tokens, size));
    withType(type, [&](auto t) {
        using T = decltype(t);
        auto launch = [&](auto own) {
            constexpr bool kOwn = decltype(own)::value;
            auto with = [&](auto bytes) {
                const auto kernel = gatedBackward<T, decltype(bytes)::value, kOwn>;
                const size_t smem = kStages * (kOwn ? 4 : 3) * kTensorBytes<T>;
                ensureDynamicSmem(reinterpret_cast<const void *>(kernel), smem);
                const int resident = residentPerSm(reinterpret_cast<const void *>(kernel), kThreads, smem) * currentDevice().sms;
                {
                    KernelTimer timer__("gatedBackward", st);
                    launchDependent(kernel, static_cast<unsigned>(std::min<int64_t>(p.tiles, resident)), kThreads, smem, st, p);
                }
                afterLaunch("gatedBackward");
            };
            withPiece<T>(piece, with);
        };
        if (p.input.data) launch(std::true_type{});
        else launch(std::false_type{});
    });
}

}  // namespace gated
}  // namespace rxmet
