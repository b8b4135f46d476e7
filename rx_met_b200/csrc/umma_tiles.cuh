// Operand tiles that TMA lays down with a 128-byte swizzle, as the tensor cores read them, and products of CTA pairs.
//
// A tile is rows of 128 bytes; 16-byte piece c of row r lies at r * 128 + ((c ^ (r & 7)) * 16), from a multiple of 1024 bytes on.  Read along its rows (K-major:
// a row is an element of M or N, its bytes run along K) a product step of 32 bytes starts 32 bytes further on in the first row.  Read across them
// (MN-major: a row is an element of K, its bytes are 64 16-bit elements of M or N) a step of 16 rows starts 2048 bytes further on.
#pragma once

#include "cluster_device.cuh"
#include "tensor_map.cuh"
#include "umma_device.cuh"

namespace rxmet {
namespace ummatiles {

using namespace umma;

// Start address >> 4 in bits [0,14), distance of eight rows (1024 bytes) >> 4 in [32,46), version 1 in [46,48), 128-byte swizzle (2) in [61,64).
// The distance of neighbouring blocks of 64 elements along MN, in [16,30), is needed by MN-major tiles of more than 64.
__device__ __forceinline__ uint64_t swizzledDescriptor(uint32_t addr, uint32_t blockStride = 16) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | (static_cast<uint64_t>((blockStride >> 4) & 0x3fffu) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

// Two- to four-dimensional boxes; `map` describes them, coordinates from the innermost outwards.
__device__ __forceinline__ void copyTile2(uint32_t to, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// The same in a CTA pair: the bytes arrive at the barrier of the pair's first CTA, whose shared-memory addresses have bit 24 clear.
__device__ __forceinline__ void copyTile2Pair(uint32_t to, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(y),
                 "r"(bar & 0xfeffffffu)
                 : "memory");
}
__device__ __forceinline__ void copyTile4(uint32_t to, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w),
                 "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void fenceAsyncProxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void prefetchMap(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

template <int CTAS>
__device__ __forceinline__ void allocTmem(uint32_t slot, uint32_t cols) {
    if constexpr (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void freeTmem(uint32_t tmem, uint32_t cols) {
    if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// kind::i8, signed codes on both sides, 32-bit integer sums: accumulator format 2 in [4,6), operand formats 1 in [7,10) and [10,13), both K-major.
__host__ __device__ constexpr uint32_t signedCodes(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void productI8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
}
// kind::f16, 32-bit sums, 128 rows of A: operand formats (0 half, 1 bfloat16) in [7,10) and [10,13); A MN-major with bit 15, B with bit 16.
__host__ __device__ constexpr uint32_t halves(bool bf16, int n, bool aMnMajor, bool bMnMajor) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (aMnMajor ? 1u << 15 : 0u) | (bMnMajor ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTileM >> 4) << 24);
}
__device__ __forceinline__ void product(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
// A in tensor memory: lane = row, a column holds two neighbours along K.
__device__ __forceinline__ void productTmem(uint32_t tmem, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tmemStoresDone() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Barrier of some of a CTA's threads.
__device__ __forceinline__ void groupBarrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// Arrives at the barrier of both CTAs of a pair once the products issued so far are complete.
__device__ __forceinline__ void commitPair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}

__device__ __forceinline__ void loadTmem16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
__device__ __forceinline__ void loadTmem8(uint32_t at, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at));
}
__device__ __forceinline__ void loadTmem32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void storeTmem16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
        "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void loadsDone() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void arriveRemote(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

}  // namespace ummatiles

// Binds the current device's context to this thread, which encoding a tensor map needs: a thread of the autograd engine may come here without one.
inline void bindContext() { RXMET_CUDA(cudaSetDevice(currentDevice().device)); }

}  // namespace rxmet
