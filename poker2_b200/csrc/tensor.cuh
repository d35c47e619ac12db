// Tensor-core plumbing of sm_100a: bounded mbarrier waits, TMA loads, tensor memory, matrix instructions.
#pragma once

#include "common.cuh"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace p2b {
namespace tc {

// A wait that takes longer than this many clocks (about two seconds) is given up: the kernel then ends with its outputs
// marked instead of holding the GPU.
constexpr long long kWaitClocks = 4000000000ll;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// True once the phase of `parity` is over; false if that took too long or another warp of the block has given up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* given_up) {
    if (mbar_try(bar, parity)) return true;
    const long long begin = clock64();
    while (!mbar_try(bar, parity)) {
        if (*given_up) return false;
        if (clock64() - begin > kWaitClocks) {
            *given_up = 1;
            return false;
        }
    }
    return true;
}

// ---- two blocks of a cluster as a pair: rank 0 leads, its barriers are told what both do ----
__device__ __forceinline__ uint32_t pair_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// the leader's barrier at the same place of its shared memory
__device__ __forceinline__ uint32_t in_leader(uint32_t bar) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(bar));
    return r;
}
// (relaxed: what the leader waits for are reads of tensor memory, over when their wait is; a release would wait for the stores
// to global memory too)
__device__ __forceinline__ void pair_arrive(uint32_t leader_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_bar) : "memory");
}
__device__ __forceinline__ bool pair_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// mbar_wait for a barrier that the other block arrives at too
__device__ __forceinline__ bool pair_wait(uint32_t bar, uint32_t parity, volatile int* given_up) {
    if (pair_try(bar, parity)) return true;
    const long long begin = clock64();
    while (!pair_try(bar, parity)) {
        if (*given_up) return false;
        if (clock64() - begin > kWaitClocks) {
            *given_up = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// After a wait that ran out: longer than any copy or matrix instruction in flight takes (tens of milliseconds).
__device__ __forceinline__ void let_settle() {
    const long long begin = clock64();
    while (clock64() - begin < 50000000ll) {
    }
}
// tma_load_2d into the own block's memory, counted by the leader's barrier
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t leader_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(leader_bar)
        : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t dst, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns) : "memory");
}
__device__ __forceinline__ void pair_tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
// what the pair's matrix instructions so far end with arrives at this barrier of both blocks
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
}
// 256 rows (128 of each block) x n columns (n / 2 operand rows in each block)
__device__ __forceinline__ void pair_mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}

// Box of a 2-D tensor at element (x, y) into shared memory; bytes outside the tensor arrive as zeros.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// `bytes` (a multiple of 16) from one 16-byte boundary to another.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// A box from shared memory to a 2-D tensor at element (x, y), both inside it; what lies outside is left out.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// until all but the last kLeft groups of stores have read their shared memory
template <int kLeft> __device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void group_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// Tensor memory: the whole warp allocates and frees; the address lands in shared memory.
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 lanes x 32 columns of 32 bits: lane l of the warp gets row l of its quadrant.
__device__ __forceinline__ void tmem_load_32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
          "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
          "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load_16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory operand, 128-byte swizzle (tiles of 8 rows x 128 bytes start on 1024-byte boundaries).
// group_stride: bytes between 8-row groups; chunk_stride: bytes between 128-byte chunks (used when the rows are not along K).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t group_stride, uint32_t chunk_stride) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(chunk_stride >> 4) << 16) | ((uint64_t)(group_stride >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// 16-bit operands, fp32 accumulator.
__host__ __device__ constexpr uint32_t f16_idesc(bool bf16, bool a_rows_along_k, bool b_rows_along_k, int m, int n) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_rows_along_k ? 1u : 0u) << 15) |
           ((b_rows_along_k ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}

}  // namespace tc

// Tensor map of a row-major matrix: boxes of `box_rows` rows x 128 bytes, 128-byte swizzle.  `element` is the size of an
// element (2: 16-bit, 1: bytes); base and stride are multiples of 16 bytes (checked by the callers with a message of their own).
int encode_rows(CUtensorMap* map, const void* base, int element, int64_t columns, int64_t rows, int64_t stride_bytes, int box_rows);
// The same of packed bytes in pieces of 1024, without a swizzle: box y = 8 * piece.
int encode_pieces(CUtensorMap* map, const void* base, int64_t pieces);

namespace tc {

// 4-bit operands (two 64-wide K halves share a 32-bit scale word), fp32 accumulator: one power-of-two scale for 32 values.
// scale words: tensor memory, lane r of each quadrant, column j = the four scales of row 32 j + r.
__host__ __device__ constexpr uint32_t mx4_idesc(int m, int n, int scale_half) {
    return ((uint32_t)(2 * scale_half) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) |
           ((uint32_t)(m >> 7) << 27) | ((uint32_t)(2 * scale_half) << 29);
}
__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b,
                                        uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(add)
        : "memory");
}
// 512 bytes of shared memory (32 rows of 16 bytes, no swizzle) to 4 columns, the same for each of the four quadrants.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (8ull << 32) | (1ull << 46);
}
// the pair's: 256 rows x n columns, the scales of its own 128 rows and of all n columns in either block's tensor memory
__host__ __device__ constexpr uint32_t pair_mx4_idesc(int n, int scale_half) {
    return ((uint32_t)(2 * scale_half) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (2u << 27) |
           ((uint32_t)(2 * scale_half) << 29);
}
__device__ __forceinline__ void pair_mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(add)
        : "memory");
}
__device__ __forceinline__ void pair_copy_scales(uint32_t dst, uint64_t src) {  // in both blocks, each from its own shared memory
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void tmem_copy_scales(uint32_t dst, uint64_t src) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(dst), "l"(src) : "memory");
}

}  // namespace tc
}  // namespace p2b
