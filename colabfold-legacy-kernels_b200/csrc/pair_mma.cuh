// tcgen05 and TMA forms for a pair of CTAs (cta_group::2): one MMA of 256 rows over the shared and
// tensor memory of both CTAs of a two-CTA cluster, issued by the even CTA (the leader). Loads carry
// no multicast: each CTA brings its own half of A and B into its own shared memory and counts it on
// the leader's barrier.
#pragma once

#include "sm100.cuh"

namespace cflk {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// the shared::cluster address of this CTA's `saddr` in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
}

// `bar`: a shared::cluster address, of a barrier in either CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                                 int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile"
        ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void mma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate));
}

// mma_ss_k4 for the pair: 256 x 256 x 16 MMAs run about 130 cycles each, which is what one took to
// issue when every step built its descriptors.
template <uint32_t A_STEP, uint32_t B_STEP>
__device__ __forceinline__ void mma_pair_k4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                            uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.u32 x, %1, %5;\n\tadd.u32 y, %2, %6;\n\t"
        "mov.b64 a, {x, %7};\n\tmov.b64 b, {y, %7};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, x, %5;\n\tadd.u32 y, y, %6;\n\t"
        "mov.b64 a, {x, %7};\n\tmov.b64 b, {y, %7};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, x, %5;\n\tadd.u32 y, y, %6;\n\t"
        "mov.b64 a, {x, %7};\n\tmov.b64 b, {y, %7};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, 1;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(A_STEP), "n"(B_STEP), "n"(kDescHi)
        : "memory");
}

// one arrive on this barrier of both CTAs once every MMA this thread issued before has completed
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst)),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}

}  // namespace cflk
