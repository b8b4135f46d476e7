// Linear attention with a decay for each head, one token: the states are read and written once.
//
// A CTA takes a head of a row of the batch, or a slice of its columns where there are few of them.  A lane holds four neighbouring columns, the lanes of a warp one or more whole
// rows of the slice, the eight warps take turns over the rows; eight rows a thread are asked for before the first is used.  The parts of q S that the warps have are added up
// in their order.  Bound: HBM: 4096 heads of 128 x 128 83 us, 6.5 TB/s, 256 heads 6.4 us (the
// kernel for several tokens 516 and 28).
#include "decayed_attention.h"
#include "dependent_launch.cuh"
#include "element_types.cuh"

namespace rxmet {
namespace decayed {
namespace {

constexpr int kWarps = 8, kAtOnce = 8;

template <class T>
__global__ void __launch_bounds__(32 * kWarps) decayedStep(const __grid_constant__ Pass p, const int columns) {
    __shared__ float sq[kMaxDim], sk[kMaxDim];
    __shared__ float4 parts[kWarps][32];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = blockIdx.z * columns, lanes = columns / 4, together = 32 / lanes;   // columns of this CTA, lanes for a row of them, rows of a warp at a time
    const int sub = lane / lanes, col = first + (lane - sub * lanes) * 4;
    const bool works = sub < together && col < p.value;
    const int stride = kWarps * together, row0 = warp * together + sub;
    waitForPredecessor();
    const bool live = !p.lengths || p.lengths[b] > 0;
    const size_t head = (static_cast<size_t>(b) * p.heads + h) * p.key * p.value;
    const float4 *in = p.stateIn ? reinterpret_cast<const float4 *>(p.stateIn + head + col) : nullptr;
    float4 *out = p.stateOut ? reinterpret_cast<float4 *>(p.stateOut + head + col) : nullptr;
    const size_t pitch = p.value / 4;

    float4 s[kAtOnce];
    auto load = [&](int from) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int row = from + i * stride;
            s[i] = works && in && row < p.key ? in[row * pitch] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    load(row0);
    auto element = [&](const rxmet_head_tensor &t, int d) {
        return toFloat(static_cast<const T *>(t.data)[b * t.stride_b + static_cast<int64_t>(h / (p.heads / t.heads)) * t.stride_h + d]);
    };
    if (live && tid < p.key) {
        sq[tid] = element(p.q, tid);
        sk[tid] = element(p.k, tid);
    }
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live && works) v = make_float4(element(p.v, col), element(p.v, col + 1), element(p.v, col + 2), element(p.v, col + 3));
    // a row of the batch without a token keeps its state
    // The decay as a sum of two floats: rounded to one, its error would grow with every token that a state remembers.
    const double exact = live ? exp(static_cast<double>(p.logDecay[h])) : 1.0;
    const float decay = static_cast<float>(exact), rest = static_cast<float>(exact - decay);
    letDependentsStart();
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int from = row0; from < p.key; from += kAtOnce * stride) {
        if (from > row0) load(from);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int row = from + i * stride;
            if (!works || row >= p.key) continue;
            if (live) {
                const float k = sk[row], q = sq[row];
                s[i].x = fmaf(s[i].x, decay, fmaf(s[i].x, rest, k * v.x));
                s[i].y = fmaf(s[i].y, decay, fmaf(s[i].y, rest, k * v.y));
                s[i].z = fmaf(s[i].z, decay, fmaf(s[i].z, rest, k * v.z));
                s[i].w = fmaf(s[i].w, decay, fmaf(s[i].w, rest, k * v.w));
                o.x = fmaf(q, s[i].x, o.x);
                o.y = fmaf(q, s[i].y, o.y);
                o.z = fmaf(q, s[i].z, o.z);
                o.w = fmaf(q, s[i].w, o.w);
            }
            if (out) out[row * pitch] = s[i];
        }
    }
    parts[warp][lane] = o;
    __syncthreads();
    for (int c = tid; c < min(columns, p.value - first); c += blockDim.x) {
        float sum = 0.f;
        for (int w = 0; w < kWarps; ++w)
            for (int i = 0; i < together; ++i) sum += reinterpret_cast<const float *>(&parts[w][i * lanes + c / 4])[c & 3];
        if (p.out) static_cast<T *>(p.out)[(static_cast<size_t>(b) * p.heads + h) * p.value + first + c] = fromFloat<T>(live ? sum * p.outScale : 0.f);
    }
}

}  // namespace

bool takesStep(const Pass &p) {
    return p.tokens == 1 && !p.reverse && !p.outFloat && p.stateCol == 1 && p.value % 4 == 0 && alignedTo(p.stateIn, 16) && alignedTo(p.stateOut, 16) && p.inScale == 1.f && p.finalScale == 1.f;
}

void launchStep(const Pass &p, int type, cudaStream_t st) {
    // slices of a head until there are CTAs for all SMs, but no less than 128 bytes of a row
    int columns = (p.value + 3) / 4 * 4;
    while (columns % 2 == 0 && columns / 2 >= 32 && columns / 2 % 4 == 0 && static_cast<int64_t>(p.heads) * p.batch * (p.value / columns) < 2 * currentDevice().sms) columns /= 2;
    const dim3 grid(p.heads, p.batch, (p.value + columns - 1) / columns);
    withType(type, [&](auto t) {
        {
            KernelTimer timer__("decayedStep", st);
            launchDependent(decayedStep<decltype(t)>, grid, 32 * kWarps, 0, st, p, columns);
        }
        afterLaunch("decayedStep");
    });
}

}  // namespace decayed
}  // namespace rxmet
