// fg_tcgen05.cuh — wrappers of the sm_100a tensor-core instructions used by the
// LM-head kernel: tensor memory, tcgen05.mma on 16-bit operands, tiled TMA loads.
#pragma once

#include <cuda.h>

#include "fg_common.cuh"

namespace fg {
namespace tc {

// CG: CTAs that issue a product together (cta_group): 1, or 2 for a pair of SMs.

// ---- tensor memory ---------------------------------------------------------
// One warp (of each CTA of the pair) allocates `cols` columns (a power of two,
// 32..512) and gives up the right to allocate more; the base address lands in
// *slot. The same warp frees.
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(cols) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Eight neighbouring fp32 columns of the warp's 32 lanes, one lane a thread.
__device__ __forceinline__ void tmem_ld8(float (&v)[8], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(addr));
}
// 16 lanes by eight columns in the layout of a warp-level product's accumulator:
// thread (g, t) gets columns 2t, 2t + 1 of lane g, then of lane g + 8.
__device__ __forceinline__ void tmem_ld_window(float (&v)[4], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(const float* v, uint32_t addr) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                 :: "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
                    "r"(addr) : "memory");
}
// The loaded registers hold their values only past the wait: tying them to it
// keeps their uses behind it.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(float (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- shared-memory operands ------------------------------------------------
// Descriptor of a K-major tile of 64 16-bit elements a row (128 bytes, 128-byte
// swizzle, 8-row groups 1024 bytes apart), the layout a 64-wide TMA box leaves.
// The next 16 elements of K start 32 bytes further (+2 in the address field).
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem) {
    return uint64_t((smem & 0x3ffffu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor: fp32 accumulator, both operands K-major, M x N.
__device__ __forceinline__ uint32_t instr_desc(int dtype, int m, int n) {
    const uint32_t fmt = dtype == FG_DTYPE_BF16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}
// D[tmem] (+)= A * B^T, K = 16; issued by one thread (of the pair's first CTA:
// each CTA of the pair then holds M / 2 rows of A, N / 2 rows of B and its own M / 2
// lanes of D, at the same addresses).
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate)) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate)) : "memory");
}
// One arrival on `bar` (of every CTA of the pair) when every mma issued so far by
// this thread has finished.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                     :: "r"(smem_u32(bar)) : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
            :: "r"(smem_u32(bar)), "h"(uint16_t(3)) : "memory");
}
// The same on this CTA's barrier alone.
template <int CG>
__device__ __forceinline__ void commit_here(uint64_t* bar) {
    if constexpr (CG == 1)
        commit<1>(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                     :: "r"(smem_u32(bar)) : "memory");
}

// ---- the pair --------------------------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Cluster address of `p`'s counterpart in CTA `rank`.
__device__ __forceinline__ uint32_t mapa(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" :: "r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(bar) : "memory");
}

// ---- TMA -------------------------------------------------------------------
// `bar` is a cluster address; with CG = 2 it may be the other CTA's.
template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3}], [%4];"
            :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3}], [%4];"
            :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(map) : "memory");
}

// ---- dependent launches ----------------------------------------------------
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace tc
}  // namespace fg
