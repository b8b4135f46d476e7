// Linear attention with a decay for each head: entry points, passes of the forward and of the gradients, sums over shared heads.
#include "decayed_attention.h"
#include "dependent_launch.cuh"
#include "element_types.cuh"

namespace rxmet {
namespace decayed {
namespace {

// out[row][g][d] = sum over the `share` heads of group g of part[row][g * share + i][d], in their order.
template <class T>
__global__ void __launch_bounds__(256) sumSharedHeads(const float *part, int64_t rows, int groups, int share, int dim, T *out) {
    waitForPredecessor();
    letDependentsStart();
    const int64_t count = rows * groups * dim;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t group = i / dim, d = i - group * dim;
        float sum = 0.f;
        for (int k = 0; k < share; ++k) sum += part[(group * share + k) * dim + d];
        out[i] = fromFloat<T>(sum);
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


}  // namespace
}  // namespace decayed
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::decayed;

extern "C" {

size_t rxmet_decayed_attention_workspace_bytes(const rxmet_decayed_attention *a, int backward) {
    WorkspaceSizer size;
    if (!a || !backward) return 0;
    const size_t rows = static_cast<size_t>(a->batch) * a->tokens * a->heads;
    if (a->q.heads != a->heads) size.take<float>(rows * a->key_dim);
    if (a->k.heads != a->heads) size.take<float>(rows * a->key_dim);
    if (a->v.heads != a->heads) size.take<float>(rows * a->value_dim);
    return size.used();
}

int rxmet_decayed_attention_forward(const rxmet_decayed_attention *problem, const float *state_dev, void *out_dev, float *final_state_dev,
                                    void *workspace_dev, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        (void)workspace_dev;
        (void)workspace_bytes;
        RXMET_REQUIRE(problem, "decayed_attention: null problem");
        const rxmet_decayed_attention &a = *problem;
        checkSizes(a);
        if (a.batch == 0) return;
        RXMET_REQUIRE(a.log_decay, "decayed_attention: null log_decay");
        Pass p = passOf(a);
        if (a.tokens > 0) roles(p, checked(a.q, a.heads, "q"), checked(a.k, a.heads, "k"), checked(a.v, a.heads, "v"), a.key_dim, a.value_dim, false, a);
        else roles(p, {nullptr, 0, 0, 0, 1}, {nullptr, 0, 0, 0, 1}, {nullptr, 0, 0, 0, 1}, a.key_dim, a.value_dim, false, a);
        p.stateIn = state_dev;
        p.stateOut = final_state_dev;
        p.out = out_dev;
        launchRecurrent(p, a.type, static_cast<cudaStream_t>(stream));
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
        RXMET_REQUIRE(a.log_decay && dout, "decayed_attention: null tensor");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        rxmet_head_tensor q{nullptr, 0, 0, 0, 1}, k = q, v = q, d = q;
        if (a.tokens > 0) {
            q = checked(a.q, a.heads, "q");
            k = checked(a.k, a.heads, "k");
            v = checked(a.v, a.heads, "v");
            d = checked(*dout, a.heads, "dout");
            RXMET_REQUIRE(d.heads == a.heads, "decayed_attention: dout has %d heads of %d", d.heads, a.heads);
        }
        Workspace ws(workspace_dev, workspace_bytes);
        const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens;
        auto run = [&](Pass p, int ownHeads, void *out) {
            p.out = out;
            if (out && ownHeads != a.heads) {
                p.out = ws.take<float>(static_cast<size_t>(rows) * a.heads * p.value);
                p.outFloat = true;
            }
            launchRecurrent(p, a.type, st);
            if (!p.outFloat || rows == 0) return;
            withType(a.type, [&](auto t) {
                using T = decltype(t);
                const int64_t count = rows * ownHeads * p.value;
                {
                    KernelTimer timer__("sumSharedHeads", st);
                    launchDependent(sumSharedHeads<T>, static_cast<unsigned>(std::min<int64_t>((count + 255) / 256, 8 * currentDevice().sms)), 256, 0, st,
                                    static_cast<const float *>(p.out), rows, ownHeads, a.heads / ownHeads, p.value, static_cast<T *>(out));
                }
                afterLaunch("sumSharedHeads");
            });
        };
        if (dq_dev) {
            Pass p = passOf(a);
            roles(p, d, v, k, a.value_dim, a.key_dim, true, a);
            p.stateIn = state_dev;
            run(p, a.q.heads, dq_dev);
        }
        if (dk_dev) {
            Pass p = passOf(a);
            roles(p, v, d, q, a.value_dim, a.key_dim, true, a);
            p.reverse = true;
            p.stateIn = dfinal_state_dev;
            p.inScale = 1.f / a.scale;
            run(p, a.k.heads, dk_dev);
        }
        if (dv_dev || dstate_dev) {
            Pass p = passOf(a);
            roles(p, k, q, d, a.key_dim, a.value_dim, false, a);
            p.reverse = true;
            p.stateIn = dfinal_state_dev;
            p.stateOut = dstate_dev;
            p.inScale = 1.f / a.scale;
            p.finalScale = a.scale;
            run(p, a.v.heads, dv_dev);
        }
    });
}

}  // extern "C"
