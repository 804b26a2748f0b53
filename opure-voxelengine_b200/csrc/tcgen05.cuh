// tcgen05.cuh -- PTX wrappers of the block-scaled tensor-core path: tiled TMA loads, tensor
// memory, and tcgen05.mma with MX operands. No TMA multicast.
#pragma once

#include <cuda.h>

#include "tma.cuh"

namespace opure {
namespace tc {

__device__ __forceinline__ void load_2d(bool one, void *dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %5, 0;\n"
        " @e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}" ::"r"(
            smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_addr(bar)), "r"(uint32_t(one))
        : "memory");
}

// Into L2 only (harmless before a dependency wait: a late write of the predecessor shows there).
__device__ __forceinline__ void prefetch_2d(bool one, const CUtensorMap *map, uint32_t x, uint32_t y) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %3, 0;\n @e cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n}" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(x), "r"(y), "r"(uint32_t(one))
        : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void alloc(uint32_t *dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// One lane of a converged warp. The loops that issue loads and MMAs run on all lanes, and the
// instructions themselves are predicated on this one (`one`): addresses and descriptors then stay
// in uniform registers, where the instructions want them, and the warp does not diverge. A loop
// inside "if (lane == 0)" moved each operand there and took 1,000 cycles for 4 MMAs that execute
// in 512; a branch around the instructions cost 150 cycles a stage to converge again.
__device__ __forceinline__ bool elect() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Descriptor of a K-major operand tile in 128-byte swizzled rows (as TMA writes it): 8-row
// groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
    return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}
// Descriptor of a scale tile: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t desc_scales(uint32_t addr) {
    return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}

// Copies a 512-byte scale tile (128 rows x 4 blocks) to 4 TMEM columns, into all four lane
// quarters: column j holds rows 32 j .., one block per byte.
__device__ __forceinline__ void copy_scales(bool one, uint32_t taddr, uint64_t desc) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %2, 0;\n @e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n}" ::"r"(taddr),
                 "l"(desc), "r"(uint32_t(one))
                 : "memory");
}

// Element formats in the instruction descriptor: of kind::mxf8f6f4, and E2M1 of kind::mxf4.
constexpr uint32_t kE4M3 = 0, kE2M1 = 5, kPackedE2M1 = 1;
// Instruction descriptor with E8M0 scales; the scale's byte (block within a column) is or'ed in.
constexpr __host__ __device__ uint32_t idesc_mx(uint32_t a_format, uint32_t b_format, uint32_t m, uint32_t n) {
    return (a_format << 7) | (b_format << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24);
}
__device__ __forceinline__ uint32_t idesc_block(uint32_t b) { return (b << 4) | (b << 29); }

// D[tmem] (+)= (A scaled) (B scaled)^T over K = 32: one scale per row.
__device__ __forceinline__ void mma_mxf8f6f4(bool one, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 e, %7, 0;\n"
        " @e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(uint32_t(one))
        : "memory");
}

// Arrives on `bar` once every tcgen05 operation this thread issued before has completed.
__device__ __forceinline__ void commit(bool one, uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
        " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_addr(bar)),
        "r"(uint32_t(one))
        : "memory");
}

// 32 neighbouring fp32 columns of this thread's TMEM lane (valid after wait_ld).
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---- CTA pairs (cta_group::2) ---------------------------------------------------------------
// The even CTA of a pair issues; D spans both CTAs' TMEM (128 rows each), each CTA's shared
// memory holds its 128 rows of A and its half of B's rows, at the same offsets in both.

// A load into this CTA that completes on an mbarrier of either CTA of the pair (a cluster address).
__device__ __forceinline__ void load_2d_pair(bool one, void *dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %5, 0;\n"
        " @e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];\n}" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "r"(uint32_t(one))
        : "memory");
}
__device__ __forceinline__ void load_4d_pair(bool one, void *dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z,
                                             uint32_t w, uint32_t bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %7, 0;\n"
        " @e cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%2, %3, %4, %5}], [%6];\n}" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar), "r"(uint32_t(one))
        : "memory");
}
__device__ __forceinline__ void alloc_pair(uint32_t *dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Scale tile to TMEM in both CTAs, each from its own shared memory.
__device__ __forceinline__ void copy_scales_pair(bool one, uint32_t taddr, uint64_t desc) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %2, 0;\n @e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n}" ::"r"(taddr),
                 "l"(desc), "r"(uint32_t(one))
                 : "memory");
}
// K = 32 of byte slots, one scale per row.
__device__ __forceinline__ void mma_mxf8f6f4_pair(bool one, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                  uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 e, %7, 0;\n"
        " @e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(uint32_t(one))
        : "memory");
}
// K = 64 of packed E2M1 on both sides, two scales per row.
__device__ __forceinline__ void mma_mxf4_pair(bool one, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 e, %7, 0;\n"
        " @e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(uint32_t(one))
        : "memory");
}
// Arrives on `bar` of both CTAs once every tcgen05 operation this thread issued before has completed.
__device__ __forceinline__ void commit_pair(bool one, uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %2, 0;\n"
        " @e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}" ::"r"(
            smem_addr(bar)),
        "h"(uint16_t(3)), "r"(uint32_t(one))
        : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void expect_tx(bool one, uint64_t *bar, uint32_t bytes) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %2, 0;\n @e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(
            smem_addr(bar)),
        "r"(bytes), "r"(uint32_t(one))
        : "memory");
}
// bulk_load_keep (tma.cuh) by one lane.
__device__ __forceinline__ void bulk(bool one, void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred e;\n setp.ne.b32 e, %4, 0;\n"
        " @e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n}" ::"r"(smem_addr(dst)),
        "l"(src), "r"(bytes), "r"(smem_addr(bar)), "r"(uint32_t(one))
        : "memory");
}

// ---- TMA stores ----------------------------------------------------------------------------
__device__ __forceinline__ void store_2d(const CUtensorMap *map, uint32_t x, uint32_t y, const void *src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(smem_addr(src))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// 4 or 8 bytes to shared memory, asynchronously.
template <uint32_t BYTES>
__device__ __forceinline__ void copy_async(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- clusters --------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// This CTA's shared-memory address as CTA `rank` of the cluster sees its own.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Four floats to another CTA's shared memory, counted by an mbarrier there (cluster addresses).
__device__ __forceinline__ void st_async_f4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
                 "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar)
                 : "memory");
}
// Shared memory to a CTA of the cluster (cluster addresses), counted by an mbarrier there. The
// source has to stay until the receiver has counted it.
__device__ __forceinline__ void bulk_send(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "r"(smem_addr(src)), "r"(bytes), "r"(bar)
                 : "memory");
}

}  // namespace tc
}  // namespace opure
