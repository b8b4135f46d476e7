// Activations kept in 8 bits, and the product of an activated gate with its partner, whose backward pass starts from such codes.
//
// A thread has eight neighbouring elements, four threads a group, whose largest magnitude they find among themselves; every array is read and written once.  The step of a group is a power of two: the
// quotient and the values are exact, so that codes do not depend on how they are worked out, and products with values can be taken in 16 bits without another rounding.
#include "kept_codes.cuh"

#include "dependent_launch.cuh"
#include "row_words.cuh"

namespace rxmet {
namespace kept {
namespace {

constexpr int kThreads = 256, kAtOnce = 2, kPer = 8;
constexpr int kMaxWidth = 131071;   // as of codes of rows

struct Codes {
    int8_t *codes, *exponents;
};
struct Pass {
    int64_t rows;
    int width, words, lowest, activation;   // words: of eight elements in a row, a multiple of four
    const void *a, *b;
    int64_t aPitch, bPitch, codesPitch;
    Codes first, second;
    void *y, *z;
};

template <class T, bool WIDE>
__device__ __forceinline__ void loadEight(const void *data, int64_t pitch, const RowWord &at, int count, float (&v)[kPer]) {
    const T *from = static_cast<const T *>(data) + static_cast<int64_t>(at.row) * pitch + at.word * kPer;
    if (WIDE && count > 0) {
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < kPer / W; ++i) {
            const Pack<T, W> p = *reinterpret_cast<const Pack<T, W> *>(from + i * W);
#pragma unroll
            for (int j = 0; j < W; ++j) v[i * W + j] = toFloat(p.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = !WIDE && i < count ? toFloat(from[i]) : 0.f;
    }
}
template <class T, bool WIDE>
__device__ __forceinline__ void storeEight(void *data, int width, const RowWord &at, int count, const float (&v)[kPer]) {
    T *to = static_cast<T *>(data) + static_cast<int64_t>(at.row) * width + at.word * kPer;
    if (WIDE && count > 0) {
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < kPer / W; ++i) {
            Pack<T, W> p;
#pragma unroll
            for (int j = 0; j < W; ++j) p.v[j] = fromFloat<T>(v[i * W + j]);
            *reinterpret_cast<Pack<T, W> *>(to + i * W) = p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (!WIDE && i < count) to[i] = fromFloat<T>(v[i]);
    }
}

// By the four threads of a group.
__device__ __forceinline__ void keepEight(const Pass &p, const Codes &to, const RowWord &at, int count, const float (&v)[kPer]) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    const unsigned group = 0xfu << (threadIdx.x & 28);
    most = max(most, __shfl_xor_sync(group, most, 1));
    most = max(most, __shfl_xor_sync(group, most, 2));
    const int e = exponentOf(most, p.lowest);
    if (count > 0) {
        uint2 codes = make_uint2(0, 0);
        if (e != kBad) {
            const float inverse = powerOf(-e);
            codes = make_uint2(codesOf(v, inverse), codesOf(v + 4, inverse));
        }
        *reinterpret_cast<uint2 *>(to.codes + static_cast<int64_t>(at.row) * p.codesPitch + at.word * kPer) = codes;
    }
    if ((threadIdx.x & 3) == 0) to.exponents[static_cast<int64_t>(at.row) * (p.words / 4) + at.word / 4] = static_cast<int8_t>(e);
}
struct Held {
    uint2 codes;
    int exponent;
};
__device__ __forceinline__ Held heldEight(const Pass &p, const Codes &from, const RowWord &at, int count) {
    Held h{make_uint2(0, 0), 0};
    if (count > 0) {
        h.codes = *reinterpret_cast<const uint2 *>(from.codes + static_cast<int64_t>(at.row) * p.codesPitch + at.word * kPer);
        h.exponent = from.exponents[static_cast<int64_t>(at.row) * (p.words / 4) + at.word / 4];
    }
    return h;
}
__device__ __forceinline__ void valuesOfEight(const Held &h, float (&v)[kPer]) {
    const float step = stepOf(h.exponent);
    valuesOf(h.codes.x, step, v);
    valuesOf(h.codes.y, step, v + 4);
}
__device__ __forceinline__ int countOf(const Pass &p, const RowWord &at) { return at.real ? min(kPer, max(0, p.width - at.word * kPer)) : 0; }

// The activation's values, and its slopes where they are wanted; one test for all elements.  Normal distribution for gelu: Phi(x) keeps its bits for x far below zero, where 1 + erf does not.
template <bool SLOPES>
__device__ __forceinline__ void activate(int activation, const float (&x)[kPer], float (&y)[kPer], float (&slope)[kPer]) {
    if (activation == RXMET_ACTIVATION_RELU) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            y[i] = x[i] < 0.f ? 0.f : x[i];   // keeps a NaN
            if (SLOPES) slope[i] = x[i] > 0.f ? 1.f : x[i] <= 0.f ? 0.f : x[i];
        }
    } else if (activation == RXMET_ACTIVATION_SILU) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float e = expf(-fabsf(x[i]));
            float most;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(most) : "f"(1.f + e));
            const float least = e * most, open = x[i] > 0.f ? most : least, shut = x[i] > 0.f ? least : most;
            y[i] = x[i] * open;
            if (SLOPES) slope[i] = fmaf(y[i], shut, open);
        }
    } else if (activation == RXMET_ACTIVATION_GELU) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float p = normcdff(x[i]);
            y[i] = x[i] * p;
            if (SLOPES) slope[i] = fmaf(x[i], 0.3989422804014327f * expf(-0.5f * x[i] * x[i]), p);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            y[i] = x[i];
            if (SLOPES) slope[i] = 1.f;
        }
    }
}

template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads) keepCodes(const __grid_constant__ Pass p) {
    waitForPredecessor();
    letDependentsStart();
    eachRowWord<kAtOnce>(p.rows, p.words, blockIdx.x, gridDim.x, [&](const RowWord(&at)[kAtOnce]) {
        float v[kAtOnce][kPer];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) loadEight<T, WIDE>(p.a, p.aPitch, at[n], countOf(p, at[n]), v[n]);
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n)
            if (at[n].real) keepEight(p, p.first, at[n], countOf(p, at[n]), v[n]);
    });
}

template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads) keptValues(const __grid_constant__ Pass p) {
    waitForPredecessor();
    letDependentsStart();
    eachRowWord<kAtOnce>(p.rows, p.words, blockIdx.x, gridDim.x, [&](const RowWord(&at)[kAtOnce]) {
        Held held[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) held[n] = heldEight(p, p.first, at[n], countOf(p, at[n]));
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            float v[kPer];
            valuesOfEight(held[n], v);
            storeEight<T, WIDE>(p.y, p.width, at[n], countOf(p, at[n]), v);
        }
    });
}

// a: gate, b: up.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads) gatedProduct(const __grid_constant__ Pass p) {
    waitForPredecessor();
    letDependentsStart();
    eachRowWord<kAtOnce>(p.rows, p.words, blockIdx.x, gridDim.x, [&](const RowWord(&at)[kAtOnce]) {
        float gate[kAtOnce][kPer], up[kAtOnce][kPer];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            loadEight<T, WIDE>(p.a, p.aPitch, at[n], countOf(p, at[n]), gate[n]);
            loadEight<T, WIDE>(p.b, p.bPitch, at[n], countOf(p, at[n]), up[n]);
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            if (!at[n].real) continue;
            const int count = countOf(p, at[n]);
            if (p.first.codes) {
                keepEight(p, p.first, at[n], count, gate[n]);
                keepEight(p, p.second, at[n], count, up[n]);
            }
            float y[kPer], slope[kPer];
            activate<false>(p.activation, gate[n], y, slope);
#pragma unroll
            for (int i = 0; i < kPer; ++i) y[i] *= up[n][i];
            storeEight<T, WIDE>(p.y, p.width, at[n], count, y);
        }
    });
}

// a: dy, y: dgate, z: dup.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads) gatedProductBackward(const __grid_constant__ Pass p) {
    waitForPredecessor();
    letDependentsStart();
    eachRowWord<kAtOnce>(p.rows, p.words, blockIdx.x, gridDim.x, [&](const RowWord(&at)[kAtOnce]) {
        float dy[kAtOnce][kPer];
        Held gates[kAtOnce], ups[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const int count = countOf(p, at[n]);
            loadEight<T, WIDE>(p.a, p.aPitch, at[n], count, dy[n]);
            gates[n] = heldEight(p, p.first, at[n], count);
            ups[n] = heldEight(p, p.second, at[n], count);
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const int count = countOf(p, at[n]);
            float gate[kPer], up[kPer], y[kPer], slope[kPer];
            valuesOfEight(gates[n], gate);
            valuesOfEight(ups[n], up);
            activate<true>(p.activation, gate, y, slope);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                y[i] *= dy[n][i];
                slope[i] *= up[i] * dy[n][i];
            }
            if (p.z) storeEight<T, WIDE>(p.z, p.width, at[n], count, y);
            if (p.y) storeEight<T, WIDE>(p.y, p.width, at[n], count, slope);
        }
    });
}

bool wideRows(const void *data, int64_t rows, int64_t pitch, size_t size) { return alignedTo(data, 16) && (rows <= 1 || pitch * static_cast<int64_t>(size) % 16 == 0); }

Pass passOf(int64_t rows, int width, int type, const char *what) {
    RXMET_REQUIRE(rows >= 0 && width >= 1, "%s: %lld rows of %d elements", what, static_cast<long long>(rows), width);
    RXMET_REQUIRE(type == RXMET_TYPE_F32 || type == RXMET_TYPE_BF16 || type == RXMET_TYPE_F16, "%s: unknown element type %d", what, type);
    if (width > kMaxWidth) fail(RXMET_ERR_UNSUPPORTED, "%s: rows of %d elements, at most %d", what, width, kMaxWidth);
    Pass p{};
    p.rows = rows;
    p.width = width;
    p.words = 4 * groupsOf(width);
    p.lowest = lowestExponent(type);
    return p;
}
void requireCodes(const Pass &p, const void *codes, const void *exponents, const char *what) {
    RXMET_REQUIRE(codes && exponents, "%s: null pointer", what);
    RXMET_REQUIRE(alignedTo(codes, 16) && p.codesPitch % 16 == 0 && (p.rows == 1 || p.codesPitch >= p.width), "%s: rows of codes must start on 16 bytes, and apart", what);
}

template <class F>
void launch(F kernel, const char *name, const Pass &p, cudaStream_t st) {
    const int blocks = rowWordBlocks(p.rows, p.words, kAtOnce, kThreads, currentDevice().sms * residentPerSm(reinterpret_cast<const void *>(kernel), kThreads, 0));
    {
        KernelTimer timer__(name, st);
        launchDependent(kernel, blocks, kThreads, 0, st, p);
    }
    afterLaunch(name);
}

}  // namespace
}  // namespace kept
}  // namespace rxmet

using namespace rxmet;

extern "C" int rxmet_keep_codes(int64_t rows, int width, int type, const void *x, int64_t x_pitch, int8_t *codes, int64_t codes_pitch, int8_t *exponents, void *stream) {
    return guarded([&] {
        kept::Pass p = kept::passOf(rows, width, type, "keep_codes");
        if (rows == 0) return;
        p.codesPitch = codes_pitch;
        RXMET_REQUIRE(x, "keep_codes: null pointer");
        kept::requireCodes(p, codes, exponents, "keep_codes");
        p.a = x;
        p.aPitch = x_pitch;
        p.first = {codes, exponents};
        const bool wide = width % 8 == 0 && kept::wideRows(x, rows, x_pitch, typeBytes(type));
        withType(type, [&](auto t) {
            using T = decltype(t);
            kept::launch(wide ? kept::keepCodes<T, true> : kept::keepCodes<T, false>, "keepCodes", p, static_cast<cudaStream_t>(stream));
        });
    });
}

extern "C" int rxmet_kept_values(int64_t rows, int width, int type, const int8_t *codes, int64_t codes_pitch, const int8_t *exponents, void *out, void *stream) {
    return guarded([&] {
        kept::Pass p = kept::passOf(rows, width, type, "kept_values");
        if (rows == 0) return;
        p.codesPitch = codes_pitch;
        RXMET_REQUIRE(out, "kept_values: null pointer");
        kept::requireCodes(p, codes, exponents, "kept_values");
        p.y = out;
        p.first = {const_cast<int8_t *>(codes), const_cast<int8_t *>(exponents)};
        const bool wide = width % 8 == 0 && alignedTo(out, 16);
        withType(type, [&](auto t) {
            using T = decltype(t);
            kept::launch(wide ? kept::keptValues<T, true> : kept::keptValues<T, false>, "keptValues", p, static_cast<cudaStream_t>(stream));
        });
    });
}

extern "C" int rxmet_gated_product(int64_t rows, int width, int type, int activation, const void *gate, int64_t gate_pitch, const void *up, int64_t up_pitch, void *y,
                                   int8_t *gate_codes, int8_t *gate_exponents, int8_t *up_codes, int8_t *up_exponents, int64_t codes_pitch, void *stream) {
    return guarded([&] {
        kept::Pass p = kept::passOf(rows, width, type, "gated_product");
        RXMET_REQUIRE(activation >= RXMET_ACTIVATION_NONE && activation <= RXMET_ACTIVATION_GELU, "gated_product: unknown activation %d", activation);
        if (rows == 0) return;
        p.activation = activation;
        p.codesPitch = codes_pitch;
        RXMET_REQUIRE(gate && up && y, "gated_product: null pointer");
        if (gate_codes || gate_exponents || up_codes || up_exponents) {
            kept::requireCodes(p, gate_codes, gate_exponents, "gated_product");
            kept::requireCodes(p, up_codes, up_exponents, "gated_product");
        }
        p.a = gate;
        p.aPitch = gate_pitch;
        p.b = up;
        p.bPitch = up_pitch;
        p.y = y;
        p.first = {gate_codes, gate_exponents};
        p.second = {up_codes, up_exponents};
        const size_t size = typeBytes(type);
        const bool wide = width % 8 == 0 && kept::wideRows(gate, rows, gate_pitch, size) && kept::wideRows(up, rows, up_pitch, size) && alignedTo(y, 16);
        withType(type, [&](auto t) {
            using T = decltype(t);
            kept::launch(wide ? kept::gatedProduct<T, true> : kept::gatedProduct<T, false>, "gatedProduct", p, static_cast<cudaStream_t>(stream));
        });
    });
}

extern "C" int rxmet_gated_product_backward(int64_t rows, int width, int type, int activation, const void *dy, int64_t dy_pitch, const int8_t *gate_codes,
                                            const int8_t *gate_exponents, const int8_t *up_codes, const int8_t *up_exponents, int64_t codes_pitch, void *dgate, void *dup, void *stream) {
    return guarded([&] {
        kept::Pass p = kept::passOf(rows, width, type, "gated_product backward");
        RXMET_REQUIRE(activation >= RXMET_ACTIVATION_NONE && activation <= RXMET_ACTIVATION_GELU, "gated_product backward: unknown activation %d", activation);
        if (rows == 0 || (!dgate && !dup)) return;
        p.activation = activation;
        p.codesPitch = codes_pitch;
        RXMET_REQUIRE(dy, "gated_product backward: null pointer");
        kept::requireCodes(p, gate_codes, gate_exponents, "gated_product backward");
        kept::requireCodes(p, up_codes, up_exponents, "gated_product backward");
        p.a = dy;
        p.aPitch = dy_pitch;
        p.y = dgate;
        p.z = dup;
        p.first = {const_cast<int8_t *>(gate_codes), const_cast<int8_t *>(gate_exponents)};
        p.second = {const_cast<int8_t *>(up_codes), const_cast<int8_t *>(up_exponents)};
        const bool wide = width % 8 == 0 && kept::wideRows(dy, rows, dy_pitch, typeBytes(type)) && alignedTo(dgate, 16) && alignedTo(dup, 16);
        withType(type, [&](auto t) {
            using T = decltype(t);
            kept::launch(wide ? kept::gatedProductBackward<T, true> : kept::gatedProductBackward<T, false>, "gatedProductBackward", p, static_cast<cudaStream_t>(stream));
        });
    });
}
