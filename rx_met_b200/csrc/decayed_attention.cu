// Linear attention with a decay for each head: entry points, passes of the forward and of the gradients, sums over shared heads.
#include "decayed_attention.h"
#include "dependent_launch.cuh"
#include "element_types.cuh"

namespace rxmet {
namespace decayed {
namespace {

// out[row][g][d] = sum over the `share` heads of group g of part[row][g * share + i][d], in their order; W elements a thread.  Bound: memory, and the latency of a thread's one round
// (6000 rows, 8 heads to 2: 64 elements a head 7.3 us by elements, 4.9 by fours; 96 elements 9.8 and 6.0).
template <class T, int W>
__global__ void __launch_bounds__(256) sumSharedHeads(const float *part, int64_t rows, int groups, int share, int dim, T *out) {
    waitForPredecessor();
    letDependentsStart();
    const int pieces = dim / W;
    const int64_t count = rows * groups * pieces;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t group = i / pieces;
        const int d = static_cast<int>(i - group * pieces) * W;
        const float *from = part + group * share * dim + d;
        float sum[W] = {};
#pragma unroll 4
        for (int k = 0; k < share; ++k, from += dim) {
            if constexpr (W == 4) {
                const float4 v = *reinterpret_cast<const float4 *>(from);
                sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
            } else sum[0] += *from;
        }
        T *to = out + group * dim + d;
        if constexpr (W == 4 && sizeof(T) == 2) *reinterpret_cast<uint2 *>(to) = make_uint2(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]));
        else if constexpr (W == 4) *reinterpret_cast<float4 *>(to) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        else *to = fromFloat<T>(sum[0]);
    }
}

rxmet_head_tensor checked(const rxmet_head_tensor &t, int heads, const char *name) {
    RXMET_REQUIRE(t.data, "decayed_attention: null %s", name);
    RXMET_REQUIRE(t.heads >= 1 && heads % t.heads == 0, "decayed_attention: %d heads of %s do not divide %d heads", t.heads, name, heads);
    return t;
}

void checkSizes(const rxmet_decayed_attention &a) {
    RXMET_REQUIRE(a.batch >= 0 && a.tokens >= 0 && a.heads >= 1 && a.key_dim >= 1 && a.value_dim >= 1,
                  "decayed_attention: batch %d, tokens %d, heads %d, key_dim %d, value_dim %d", a.batch, a.tokens, a.heads, a.key_dim, a.value_dim);
    if (a.key_dim > kMaxDim || a.value_dim > kMaxDim)
        fail(RXMET_ERR_UNSUPPORTED, "decayed_attention: heads of %d and %d elements, at most %d", a.key_dim, a.value_dim, kMaxDim);
    if (a.tokens > kMaxTokens) fail(RXMET_ERR_UNSUPPORTED, "decayed_attention: %d tokens, at most %d", a.tokens, kMaxTokens);
    if (a.batch > 65535 || a.heads > 65535) fail(RXMET_ERR_UNSUPPORTED, "decayed_attention: batch %d, heads %d, at most 65535 each", a.batch, a.heads);
    RXMET_REQUIRE(a.type >= 0 && a.type <= 2, "decayed_attention: unknown element type %d", a.type);
    RXMET_REQUIRE(std::isfinite(a.scale) && a.scale != 0.f, "decayed_attention: scale has to be finite and not zero");
}

Pass passOf(const rxmet_decayed_attention &a) {
    Pass p{};
    p.batch = a.batch;
    p.tokens = a.tokens;
    p.heads = a.heads;
    p.logDecay = a.log_decay;
    p.lengths = a.lengths;
    p.outScale = a.scale;
    p.inScale = p.finalScale = 1.f;
    return p;
}
void roles(Pass &p, const rxmet_head_tensor &q, const rxmet_head_tensor &k, const rxmet_head_tensor &v, int key, int value, bool transposed, const rxmet_decayed_attention &a) {
    p.q = q;
    p.k = k;
    p.v = v;
    p.key = key;
    p.value = value;
    p.stateRow = transposed ? 1 : a.value_dim;
    p.stateCol = transposed ? a.value_dim : 1;
}


// Passes of the gradients.
Pass queryPass(const rxmet_decayed_attention &a, const rxmet_head_tensor &q, const rxmet_head_tensor &k, const rxmet_head_tensor &v, const rxmet_head_tensor &d) {
    Pass p = passOf(a);
    roles(p, d, v, k, a.value_dim, a.key_dim, true, a);
    return p;
}
Pass keyPass(const rxmet_decayed_attention &a, const rxmet_head_tensor &q, const rxmet_head_tensor &k, const rxmet_head_tensor &v, const rxmet_head_tensor &d) {
    Pass p = passOf(a);
    roles(p, v, d, q, a.value_dim, a.key_dim, true, a);
    p.reverse = true;
    p.inScale = 1.f / a.scale;
    return p;
}
Pass valuePass(const rxmet_decayed_attention &a, const rxmet_head_tensor &q, const rxmet_head_tensor &k, const rxmet_head_tensor &v, const rxmet_head_tensor &d) {
    Pass p = passOf(a);
    roles(p, k, q, d, a.key_dim, a.value_dim, false, a);
    p.reverse = true;
    p.inScale = 1.f / a.scale;
    p.finalScale = a.scale;
    return p;
}
Pass forwardPass(const rxmet_decayed_attention &a) {
    Pass p = passOf(a);
    roles(p, a.q, a.k, a.v, a.key_dim, a.value_dim, false, a);
    return p;
}

// Lanes that were forked from a stream, joined to it in the end whether or not a launch in between has failed: the caller frees what they write.
struct ForkedLanes {
    cudaStream_t stream;
    OverlapLane *lanes[3] = {};
    cudaError_t join() {
        cudaError_t first = cudaSuccess;
        for (OverlapLane *&lane : lanes) {
            if (!lane) continue;
            for (const cudaError_t error : {cudaEventRecord(lane->done[0], lane->stream), cudaStreamWaitEvent(stream, lane->done[0], 0)})
                if (first == cudaSuccess) first = error;
            lane = nullptr;
        }
        return first;
    }
    ~ForkedLanes() { join(); }
};

// Kernels by size and type.  Single tokens have a kernel of their own, chunks are taken from 16 or 32 tokens on (planChunks); tensors that TMA cannot copy, 32-bit ones and those without one of the three go token by token.
void launchPass(const Pass &p, int type, float *states, cudaStream_t st) {
    const ChunkPlan plan = planChunks(p, type);
    const bool complete = p.q.data && p.k.data && p.v.data;   // else one is all zeros
    if (complete && takesStep(p)) launchStep(p, type, st);
    else if (complete && plan.taken && chunksCanCopy(p)) launchChunks(p, type, plan, states, st);
    else launchRecurrent(p, type, st);
}

}  // namespace
}  // namespace decayed
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::decayed;

extern "C" {

size_t rxmet_decayed_attention_workspace_bytes(const rxmet_decayed_attention *a, int backward) {
    WorkspaceSizer size;
    if (!a || a->batch <= 0 || a->tokens <= 0) return 0;
    const int status = guarded([&] {
        const rxmet_head_tensor none{};
        auto states = [&](const Pass &p) {
            if (const size_t floats = planChunks(p, a->type).stateFloats(p)) size.take<float>(floats);
        };
        if (!backward) {
            states(forwardPass(*a));
            return;
        }
        for (const Pass &p : {queryPass(*a, none, none, none, none), keyPass(*a, none, none, none, none), valuePass(*a, none, none, none, none)}) states(p);
        const size_t rows = static_cast<size_t>(a->batch) * a->tokens * a->heads;
        if (a->q.heads != a->heads) size.take<float>(rows * a->key_dim);
        if (a->k.heads != a->heads) size.take<float>(rows * a->key_dim);
        if (a->v.heads != a->heads) size.take<float>(rows * a->value_dim);
    });
    return status == RXMET_OK ? size.used() : 0;
}

int rxmet_decayed_attention_forward(const rxmet_decayed_attention *problem, const float *state_dev, void *out_dev, float *final_state_dev,
                                    void *workspace_dev, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        RXMET_REQUIRE(problem, "decayed_attention: null problem");
        const rxmet_decayed_attention &a = *problem;
        checkSizes(a);
        if (a.batch == 0) return;
        RXMET_REQUIRE(a.log_decay, "decayed_attention: null log_decay");
        if (a.tokens > 0) {
            checked(a.q, a.heads, "q");
            checked(a.k, a.heads, "k");
            checked(a.v, a.heads, "v");
        }
        Pass p = forwardPass(a);
        if (a.tokens == 0) p.q = p.k = p.v = {nullptr, 0, 0, 0, 1};
        p.stateIn = state_dev;
        p.stateOut = final_state_dev;
        p.out = out_dev;
        Workspace ws(workspace_dev, workspace_bytes);
        const size_t states = planChunks(p, a.type).stateFloats(p);
        launchPass(p, a.type, states > 0 ? ws.take<float>(states) : nullptr, static_cast<cudaStream_t>(stream));
    });
}

int rxmet_decayed_attention_backward(const rxmet_decayed_attention *problem, const float *state_dev, const rxmet_head_tensor *dout,
                                     const float *dfinal_state_dev, void *dq_dev, void *dk_dev, void *dv_dev, float *dstate_dev,
                                     void *workspace_dev, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        RXMET_REQUIRE(problem, "decayed_attention: null problem");
        const rxmet_decayed_attention &a = *problem;
        checkSizes(a);
        if (a.batch == 0) return;
        RXMET_REQUIRE(a.log_decay, "decayed_attention: null log_decay");
        const bool fromOutputs = dout && dout->data && a.tokens > 0;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        rxmet_head_tensor q{nullptr, 0, 0, 0, 1}, k = q, v = q, d = q;
        if (a.tokens > 0) {
            q = checked(a.q, a.heads, "q");
            k = checked(a.k, a.heads, "k");
            v = checked(a.v, a.heads, "v");
            d.heads = a.heads;
            if (fromOutputs) {
                d = checked(*dout, a.heads, "dout");
                RXMET_REQUIRE(d.heads == a.heads, "decayed_attention: dout has %d heads of %d", d.heads, a.heads);
            } else if (dq_dev) {   // the gradient of the final state alone does not reach the queries
                RXMET_CUDA(cudaMemsetAsync(dq_dev, 0, static_cast<size_t>(a.batch) * a.tokens * q.heads * a.key_dim * typeBytes(a.type), st));
            }
        }
        const Pass passes[] = {queryPass(a, q, k, v, d), keyPass(a, q, k, v, d), valuePass(a, q, k, v, d)};
        Workspace ws(workspace_dev, workspace_bytes);
        float *states[3] = {};
        for (int i = 0; i < 3; ++i)
            if (const size_t floats = planChunks(passes[i], a.type).stateFloats(passes[i])) states[i] = ws.take<float>(floats);
        const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens;
        auto run = [&](Pass p, float *states, int ownHeads, void *out, cudaStream_t st) {
            p.out = out;
            if (out && ownHeads != a.heads) {
                p.out = ws.take<float>(static_cast<size_t>(rows) * a.heads * p.value);
                p.outFloat = true;
            }
            launchPass(p, a.type, states, st);
            if (!p.outFloat || rows == 0) return;
            withType(a.type, [&](auto t) {
                using T = decltype(t);
                const bool fours = p.value % 4 == 0 && alignedTo(out, 4 * sizeof(T));
                const int64_t count = rows * ownHeads * p.value / (fours ? 4 : 1);
                {
                    KernelTimer timer__("sumSharedHeads", st);
                    launchDependent(fours ? sumSharedHeads<T, 4> : sumSharedHeads<T, 1>, static_cast<unsigned>(std::min<int64_t>((count + 255) / 256, 8 * currentDevice().sms)), 256, 0, st,
                                    static_cast<const float *>(p.out), rows, ownHeads, a.heads / ownHeads, p.value, static_cast<T *>(out));
                }
                afterLaunch("sumSharedHeads");
            });
        };
        // The passes run side by side, because none fills the GPU with few heads; those that may have heads to sum begin.  Forward and gradients of 2 x 1024 tokens and 16 heads of 64 take 55 us
        // with two passes one after another beside the third, 40 so; of 6 x 1000 tokens, 8 heads and shared keys 104 and 88; of 8 x 2048 tokens and 16 heads, which fill it, 128 both ways.
        const bool wanted[] = {dq_dev && (fromOutputs || a.tokens == 0), dk_dev != nullptr, dv_dev || dstate_dev};
        ForkedLanes forked{st};   // the last of the passes has the caller's stream
        auto &lanes = forked.lanes;
        for (int i = 2, last = wanted[0] ? 0 : wanted[1] ? 1 : 2; i > last; --i)
            if (wanted[i]) lanes[i] = &overlapLane(i - 1);
        for (OverlapLane *lane : lanes)
            if (lane) {
                RXMET_CUDA(cudaEventRecord(lane->fork[0], st));
                RXMET_CUDA(cudaStreamWaitEvent(lane->stream, lane->fork[0], 0));
            }
        if (wanted[2]) {
            Pass p = passes[2];
            p.stateIn = dfinal_state_dev;
            p.stateOut = dstate_dev;
            run(p, states[2], a.v.heads, dv_dev, lanes[2] ? lanes[2]->stream : st);
        }
        if (wanted[1]) {
            Pass p = passes[1];
            p.stateIn = dfinal_state_dev;
            run(p, states[1], a.k.heads, dk_dev, lanes[1] ? lanes[1]->stream : st);
        }
        if (wanted[0]) {
            Pass p = passes[0];
            p.stateIn = state_dev;
            run(p, states[0], a.q.heads, dq_dev, st);
        }
        RXMET_CUDA(forked.join());
    });
}

}  // extern "C"
