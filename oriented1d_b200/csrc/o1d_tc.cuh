// The 5th-generation tensor core, TMA and mbarrier instructions that the matrix-product kernels are made of.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace o1d {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- mbarrier ---------------------------------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// (cluster scope: some of the arrivals come from the other CTA of a pair)
__device__ __forceinline__ bool bar_poll(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return done != 0;
}
// The address of a CTA's variable in CTA `rank` of its cluster.
__device__ __forceinline__ uint32_t in_cta(const void *p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void bar_arrive_in(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %cluster_ctarank;" : "=r"(r)); return r; }
// Every thread of both CTAs.
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Every wait has a limit of two seconds, thousands of times what a tile takes.  Running out raises the device flag and
// `dead`, which ends the other waits of the CTA.
constexpr unsigned long long kWaitNs = 2000000000ull;
__device__ __forceinline__ unsigned long long now_ns() { unsigned long long t; asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t)); return t; }
__device__ __noinline__ bool bar_wait_long(uint64_t *bar, uint32_t parity, volatile int *dead, int *err_flag) {
    const unsigned long long start = now_ns();
    while (now_ns() - start < kWaitNs) {
        for (int i = 0; i < 64; i++)
            if (bar_poll(bar, parity)) return true;
        if (*dead) return false;
    }
    *dead = 1;
    *err_flag = 1;
    return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *dead, int *err_flag) {
#pragma unroll 1
    for (int i = 0; i < 64; i++)
        if (bar_poll(bar, parity)) return true;
    return bar_wait_long(bar, parity, dead, err_flag);
}
// The end of a CTA that gave up: waits (with the same limit) for what it has in flight.
__device__ __forceinline__ void bar_drain(uint64_t *bar, uint32_t parity) {
    const unsigned long long start = now_ns();
    while (!bar_poll(bar, parity) && now_ns() - start < kWaitNs) {}
}

// ---- TMA --------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load3(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
                 "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
// The same for one CTA of a pair: the bytes are counted by a barrier of the pair's first CTA (`bar`: its address there).
__device__ __forceinline__ void tma_load3_pair(void *dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                     smem_addr(dst)),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---- tcgen05 ----------------------------------------------------------------------------------------
// PAIR: two CTAs of a cluster work on one tile of twice the rows; each holds its half of both operands and of the accumulator,
// and the first one's thread issues the products for both.
template <bool PAIR> __device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t cols) {      // one whole warp (of each CTA)
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <bool PAIR> __device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {        // the same warp
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Descriptor of an operand tile in shared memory, 128-byte swizzle as TMA writes it.  K-major: rows of 64 two-byte
// elements of K, eight rows an atom, `outer` = bytes between atoms (1024).  MN-major: rows of 64 elements along M or N,
// one row per k; `outer` = bytes between groups of eight k (1024), `inner` = bytes between tiles of 64 along M or N.
__device__ __forceinline__ uint64_t operand(const void *p, uint32_t inner, uint32_t outer) {
    return (uint64_t)((smem_addr(p) & 0x3ffffu) >> 4) | (uint64_t)(inner >> 4) << 16 | (uint64_t)(outer >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// bf16 x bf16 -> fp32
__host__ __device__ constexpr uint32_t instruction(int m, int n, bool a_mn, bool b_mn) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
template <bool PAIR> __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {      // one thread
    if constexpr (PAIR)
        asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b),
                     "r"(instr), "r"((uint32_t)add)
                     : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b),
                     "r"(instr), "r"((uint32_t)add)
                     : "memory");
}
// The barrier (of a pair: the one at this place in either CTA) gets one arrival when every product this thread has issued so
// far is done.
template <bool PAIR> __device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// 32 columns of the warp's 32 accumulator rows: register i of a lane is column i of its row.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(addr));
}
// The registers of earlier loads are valid behind this (they are named so that no use of them moves before it).
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

}  // namespace tc
}  // namespace o1d
