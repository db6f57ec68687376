// fz_pair.cuh -- pairs of CTAs (clusters of two whose tcgen05 operations are cta_group::2): commits to both CTAs, arrivals
// on the first CTA's barriers, tensor-memory stores.
#pragma once

#include "fz_tcgen05.cuh"

namespace zf::nerf_mlp {

// whether the phase with the given parity has completed, without waiting
__device__ __forceinline__ bool test_phase(const uint32_t bar, const uint32_t parity) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}

// the pair's MMAs issued so far arrive on both CTAs' barriers at this offset when they are done
__device__ __forceinline__ void commit_pair(const uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}

// the address of the pair's first CTA's shared memory at this offset
__device__ __forceinline__ uint32_t of_first_cta(const uint32_t address) {
    uint32_t out;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(out) : "r"(address));
    return out;
}

// an arrival on the first CTA's barrier. What it announces lies in the arriving CTA's own tensor memory or shared memory
// and is read there by the pair's MMAs: fence_before_sync or fence_async_shared before it orders that. A release at cluster
// scope would wait for this thread's global accesses as well (about 1,000 cycles measured, which bound a pipeline stage).
__device__ __forceinline__ void arrive_first_cta(const uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(of_first_cta(bar)) : "memory");
}

__device__ __forceinline__ void sync_cluster() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 16 consecutive tensor-memory columns of this thread's lane (no wait)
__device__ __forceinline__ void store_columns(const uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}

}  // namespace zf::nerf_mlp
