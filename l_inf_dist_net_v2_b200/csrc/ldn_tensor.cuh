// What kernels on the tensor cores share: tensor memory, commits, waits and arrivals within a cluster, operands' descriptors.
#pragma once
#include "ldn_head.cuh"

namespace ldn {
namespace {

constexpr int kStoreWarps = 8;             // two for each quarter of the lanes, with half of the columns each
constexpr int kProductThreads = 64 + 32 * kStoreWarps;  // a warp loads, a warp multiplies

// ---- tcgen05 -----------------------------------------------------------------------------------------------------------------
template <int CTAS>
__device__ __forceinline__ void tensor_alloc(uint32_t* slot, int columns) {
    if constexpr (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void tensor_free(uint32_t base, int columns) {
    if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
// Arrival on the barrier (of both CTAs of a pair) when the products issued so far are done
template <int CTAS>
__device__ __forceinline__ void arrive_when_done(uint64_t* bar) {
    if constexpr (CTAS == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"(static_cast<uint16_t>(3))
                     : "memory");
}
__device__ __forceinline__ void tensor_load16(uint32_t addr, int (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
// (the registers are operands, so that nothing that uses them moves in front of the wait)
__device__ __forceinline__ void tensor_load_wait(int (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                   "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// the address of this CTA's `p` in the memory of another CTA of the cluster
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// `bytes` of this CTA's shared memory to another's, counted on a barrier there
__device__ __forceinline__ void copy_to_cta(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "r"(smem_u32(src)), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait_bounded_cluster(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kMaxPolls; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if (i >= kFastPolls) __nanosleep(64);
    }
    return false;
}
// Operand in shared memory: rows of 128 bytes in groups of 8 (1024 bytes apart), 128-byte swizzle; 32 terms further is 2 more
__device__ __forceinline__ uint64_t operand(const void* p) {
    return static_cast<uint64_t>((smem_u32(p) & 0x3ffffu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// Results leave the L2 cache first: the operands are read again
template <class T>
__device__ __forceinline__ void store_once(T* p, T v) {
    if constexpr (sizeof(T) == 4) __stcs(p, v);
    else __stcs(reinterpret_cast<unsigned short*>(p), *reinterpret_cast<const unsigned short*>(&v));
}
// Place in a ring of N stages, and the parity of its turn: counted, as one thread issues a stage's work and has 500 clocks for it (with
// a tile's place found by two divisions per stage, 10000 tokens of 5120 -> 5120 took 190 us instead of 147)
template <int N>
struct RingPlace {
    int stage = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++stage == N) {
            stage = 0;
            parity ^= 1;
        }
    }
};

}  // namespace
}  // namespace ldn
