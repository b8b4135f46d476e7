// Gated linear recurrence: what its passes share.
//
// A tile is the channels of a warp's row (128 bytes of 16-bit types and of floats) times kChunk tokens of a sequence; each of a CTA's eight warps has kSteps neighbouring tokens.  A run of
// tokens maps the state before it to the one behind it by h -> A h + B, so that the warps' (A, B), joined in order, give the tile's, and the tiles' of a sequence the state in front of each of
// them: `Chain`.  The CTAs walk over tiles in the order of tickets, the first tiles of all sequences before the second ones, and a stage of shared memory is filled for the tile to come
// while one is worked on.
#pragma once

#include "cluster_device.cuh"
#include "dependent_launch.cuh"
#include "element_types.cuh"
#include "rxmet_b200_gated.h"

namespace rxmet {
namespace gated {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kSteps = 16, kChunk = kWarps * kSteps;
constexpr int kWindow = 32;                    // tiles that a look back spans
constexpr uint32_t kPollLimit = 1u << 18;      // 0.2 s of polling; a legitimate wait lasts microseconds

template <class T>
constexpr int kChannels = 128 / static_cast<int>(sizeof(T));   // of a tile
template <class T>
constexpr uint32_t kTensorBytes = kChunk * kChannels<T> * sizeof(T);   // of a tile
template <class T>
constexpr int kLane = kChannels<T> / 32;

// What the tiles of a sequence tell one another.  `parts`: (A, B) of a tile, `whole`: the state behind it; `flags` says which of them is there (1, 2).
// A state behind a tile is always A times the state in front plus B, whether one tile took that step or a later one did after looking back over several, so that bits do not depend on who was first.
struct Chain {
    unsigned *ticket;
    int *flags;       // [slab][place in the chain]
    float2 *parts;    // [slab][place][channels]
    float *whole;
    int *status;
};

struct Pass {
    int batch, tokens, width, chunks, slabsOfRow, tanhValue;
    bool paired;   // two neighbours of a 16-bit output can be written at once
    int64_t tiles;
    rxmet_token_tensor forget, value, input, dout;
    const int32_t *lengths;
    const float *state, *dfinal;
    void *out, *dforget, *dvalue, *dinput;
    float *finalState, *dstate, *marks;
    Chain chain;
};

__device__ __forceinline__ int loadFlag(const int *at) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
    return v;
}
__device__ __forceinline__ void storeFlag(int *at, int v) { asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(at), "r"(v) : "memory"); }

// sigmoid(x) = 1 - sigmoid(-x) from the smaller of the two, so that neither loses bits to a subtraction from one.
struct Gate {
    float open, shut;
    __device__ __forceinline__ explicit Gate(float x) {
        const float e = expf(-fabsf(x));
        float most;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(most) : "f"(1.f + e));   // one unit in the last place; the argument is in [1, 2]
        const float least = e * most;
        open = x > 0.f ? most : least;
        shut = x > 0.f ? least : most;
    }
};

// Copies of PIECE bytes from a row of channels to shared memory, `bytes` of them real and the rest zeros.
template <int PIECE>
__device__ __forceinline__ void copyPiece(uint32_t to, const void *from, int bytes) {
    if constexpr (PIECE == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(PIECE), "r"(bytes) : "memory");
}
__device__ __forceinline__ void commitCopies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copiesArrived() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Where a tile lies.
template <class T>
struct Tile {
    int64_t slab;
    int chunk, b, d0, live, first;   // live: of its tokens, those of the sequence; first: its first token
    __device__ __forceinline__ Tile(const Pass &p, int64_t index, bool reverse) {
        const int64_t slabs = static_cast<int64_t>(p.batch) * p.slabsOfRow;
        const int place = static_cast<int>(index / slabs);
        slab = index - place * slabs;
        chunk = reverse ? p.chunks - 1 - place : place;
        b = static_cast<int>(slab / p.slabsOfRow);
        d0 = static_cast<int>(slab - static_cast<int64_t>(b) * p.slabsOfRow) * kChannels<T>;
        first = chunk * kChunk;
        const int length = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
        live = min(max(length - first, 0), kChunk);
    }
};

// Asks for the live tokens of a tile's rows of one tensor.  A row of shared memory holds the tile's channels of one token.
template <class T, int PIECE>
__device__ __forceinline__ void askFor(uint32_t to, const rxmet_token_tensor &t, const Tile<T> &tile, int width) {
    constexpr int kRow = kChannels<T> * sizeof(T), kPieces = kRow / PIECE, kPer = PIECE / static_cast<int>(sizeof(T));
    const int r0 = threadIdx.x / kPieces, piece = threadIdx.x % kPieces;
    const int real = min(kPer, width - tile.d0 - piece * kPer);
    if (real <= 0) return;
    constexpr int kRows = kThreads / kPieces;
    const T *from = static_cast<const T *>(t.data) + tile.b * t.stride_b + (static_cast<int64_t>(tile.first) + r0) * t.stride_t + tile.d0 + piece * kPer;
    const int64_t step = kRows * t.stride_t;
    uint32_t at = to + r0 * kRow + piece * PIECE;
    for (int r = r0; r < tile.live; r += kRows, from += step, at += kRows * kRow) {
        if constexpr (PIECE >= 4) copyPiece<PIECE>(at, from, real * static_cast<int>(sizeof(T)));
        else {
            const uint16_t v = *reinterpret_cast<const uint16_t *>(from);   // rows that no asynchronous copy can take
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(v) : "memory");
        }
    }
}

// The lane's channels of a row.
template <class T>
__device__ __forceinline__ void readRow(const uint8_t *row, float (&v)[kLane<T>]) {
    if constexpr (sizeof(T) == 4) v[0] = *reinterpret_cast<const float *>(row);
    else {
        const float2 two = unpack2<T>(*reinterpret_cast<const uint32_t *>(row));
        v[0] = two.x;
        v[1] = two.y;
    }
}
template <class T>
__device__ __forceinline__ void writeRow(T *to, const float (&v)[kLane<T>], int real, bool paired) {
    if constexpr (sizeof(T) == 4) {
        if (real > 0) *to = v[0];
    } else {
        if (paired) {
            if (real > 0) *reinterpret_cast<uint32_t *>(to) = pack2<T>(v[0], v[1]);
        } else {
            if (real > 0) to[0] = fromFloat<T>(v[0]);
            if (real > 1) to[1] = fromFloat<T>(v[1]);
        }
    }
}

// The state in front of the tile at `place` of its chain, for the lane's channels.  All threads of the CTA; the predecessors hold lower tickets, whose CTAs are at work already, so that the
// wait ends.  One warp polls the flags of the last kWindow tiles until the nearest state and every (A, B) behind it are there.
template <int N>
__device__ __forceinline__ void stateBefore(const Chain &c, int64_t slab, int place, int chunks, float2 (*window)[32 * N], int *nearest, float (&h)[N]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t base = slab * chunks + place - 1;
    if (warp == 0) {
        int found = -1;
        for (uint32_t poll = 0; poll < kPollLimit && found < 0; ++poll) {
            const int flag = place - 1 - lane >= 0 ? loadFlag(c.flags + base - lane) : 0;
            const unsigned whole = __ballot_sync(0xffffffffu, flag == 2), some = __ballot_sync(0xffffffffu, flag != 0);
            if (whole) {
                const int at = __ffs(whole) - 1;
                const unsigned nearer = (1u << at) - 1;
                if ((some & nearer) == nearer) found = at;
            }
        }
        if (lane == 0) {
            if (found < 0) atomicExch(c.status, 1);
            *nearest = found;
        }
    }
    __syncthreads();
    const int back = max(*nearest, 0);
    for (int i = warp; i < back; i += kWarps)
#pragma unroll
        for (int v = 0; v < N; ++v) window[i][lane * N + v] = __ldcg(c.parts + (base - i) * (32 * N) + lane * N + v);
#pragma unroll
    for (int v = 0; v < N; ++v) h[v] = __ldcg(c.whole + (base - back) * (32 * N) + lane * N + v);
    if (back == 0) return;
    __syncthreads();
    for (int i = back - 1; i >= 0; --i)
#pragma unroll
        for (int v = 0; v < N; ++v) {
            const float2 part = window[i][lane * N + v];
            h[v] = fmaf(part.x, h[v], part.y);
        }
}
// By one warp: the tile's (A, B), or the state behind it.
template <int N>
__device__ __forceinline__ void tellPart(const Chain &c, int64_t at, const float (&a)[N], const float (&b)[N]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int v = 0; v < N; ++v) __stcg(c.parts + at * (32 * N) + lane * N + v, make_float2(a[v], b[v]));
    __threadfence();
    __syncwarp();
    if (lane == 0) storeFlag(c.flags + at, 1);
}
template <int N>
__device__ __forceinline__ void tellWhole(const Chain &c, int64_t at, const float (&h)[N]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int v = 0; v < N; ++v) __stcg(c.whole + at * (32 * N) + lane * N + v, h[v]);
    __threadfence();
    __syncwarp();
    if (lane == 0) storeFlag(c.flags + at, 2);
}

// The tiles of a CTA: by tickets where tiles wait for one another, else every gridDim.x'th.  `take` is called by one thread, once for each tile.
struct Tickets {
    const Pass &p;
    int64_t next;
    __device__ __forceinline__ explicit Tickets(const Pass &pass) : p(pass), next(blockIdx.x) {}
    __device__ __forceinline__ int64_t take() {
        if (p.chunks > 1) return atomicAdd(p.chain.ticket, 1u);
        const int64_t now = next;
        next += gridDim.x;
        return now;
    }
};

// Bytes that copies of a tensor's rows can take at once: 16, 4 or one element.
inline int pieceOf(const rxmet_token_tensor &t, int batch, int tokens, size_t size) {
    auto fits = [&](int bytes) {
        return alignedTo(t.data, bytes) && (batch == 1 || t.stride_b * static_cast<int64_t>(size) % bytes == 0) && (tokens == 1 || t.stride_t * static_cast<int64_t>(size) % bytes == 0);
    };
    return fits(16) ? 16 : fits(4) ? 4 : 2;
}
// f(size of a copy) for the rows' alignment.
template <class T, class F>
void withPiece(int piece, F f) {
    if (piece == 16) f(std::integral_constant<int, 16>{});
    else if (piece == 4 || sizeof(T) == 4) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, sizeof(T) == 4 ? 4 : 2>{});
}

// Launches of gated_recurrence.cu and gated_recurrence_backward.cu.
void launchForward(const Pass &p, int type, cudaStream_t st);
void launchBackward(const Pass &p, int type, cudaStream_t st);

}  // namespace gated
}  // namespace rxmet
