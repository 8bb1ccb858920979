// The integer product on the tensor cores: tcgen05.mma of 8-bit integers, operands by TMA, 32-bit sums in tensor memory.
//
// The weight is the operand whose rows are the accumulator's lanes and the tokens are its columns, so that a tile can be as narrow
// as there are tokens, and a warp's 32 lanes store 32 neighbouring outputs of one token.  Rows are read 128 terms at a time (the
// 128-byte swizzle's width); what lies outside the operands arrives as zeros.
//
// Bound by the tensor pipe where there are many tokens (10000, 5120 -> 5120: 147 us, 3.6 POP/s, of 8180 multiply-adds per clock and SM
// that the instruction takes), by start, fill and drain where there are few (512, 5120 -> 2048: 10 us).
#pragma once
#include "ldn_head.cuh"
#include "ldn_int8.cuh"

namespace ldn {
namespace {

constexpr int kTerms = 128;                // per stage
constexpr int kLanes = 128;                // outputs per CTA
constexpr int kLaneBytes = kLanes * kTerms;
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
template <int CTAS>
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                     "l"(a), "l"(b), "r"(kind), "r"(static_cast<uint32_t>(add))
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                     "l"(a), "l"(b), "r"(kind), "r"(static_cast<uint32_t>(add))
                     : "memory");
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
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int k, int row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(k), "r"(row)
        : "memory");
}
// The same into this CTA's memory, counted on a barrier of the pair's first CTA (`bar` is its address there)
__device__ __forceinline__ void load_tile_of_pair(void* dst, const CUtensorMap* map, uint32_t bar, int k, int row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(row)
        : "memory");
}
// Operand in shared memory: rows of 128 bytes in groups of 8 (1024 bytes apart), 128-byte swizzle; 32 terms further is 2 more
__device__ __forceinline__ uint64_t operand(const void* p) {
    return static_cast<uint64_t>((smem_u32(p) & 0x3ffffu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// signed 8-bit x signed 8-bit -> 32-bit integers, both operands with neighbouring terms next to each other
__host__ __device__ constexpr uint32_t product_kind(int rows, int columns) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(columns >> 3) << 17) | (static_cast<uint32_t>(rows >> 4) << 24);
}

// Results leave the L2 cache first: the operands are read again
template <class T>
__device__ __forceinline__ void store_once(T* p, T v) {
    if constexpr (sizeof(T) == 4) __stcs(p, v);
    else __stcs(reinterpret_cast<unsigned short*>(p), *reinterpret_cast<const unsigned short*>(&v));
}
// What follows the sums: a thread has one output of 16 tokens at a time, the first of them at `to`, `columns` of them there; the
// tokens' scales lie in shared memory.
template <class T>
__device__ __forceinline__ void store16(const ProductArgs& a, const int (&sum)[16], const float* scales, float w_scale, float bias,
                                        int columns, bool there, T* to) {
    float v[16], scale[16];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
        const float4 s = *reinterpret_cast<const float4*>(scales + j);
        scale[j] = s.x; scale[j + 1] = s.y; scale[j + 2] = s.z; scale[j + 3] = s.w;
    }
    product_values(sum, scale, w_scale, bias, a.activation, v);
    char* p = reinterpret_cast<char*>(to);
    const size_t row = static_cast<size_t>(a.N) * sizeof(T);  // (15 rows of 72 million outputs are more than 32 bits count)
    if (there && columns >= 16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) store_once(reinterpret_cast<T*>(p + j * row), from_float<T>(v[j]));
    } else if (there) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < columns) store_once(reinterpret_cast<T*>(p + j * row), from_float<T>(v[j]));
    }
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

// ---- tiles of 128 outputs x TOKENS, the terms split over a cluster ----------------------------------------------------------------
// For up to some hundred tokens the weight's bytes are what takes the time, and there are fewer tiles than SMs: up to eight CTAs of
// a cluster have a share of the terms each, and add their integer sums up in shared memory, in which no order shows.
__host__ __device__ constexpr int stages_of(int tokens) { return tokens == 256 ? 4 : tokens == 128 ? 6 : 8; }
__host__ __device__ constexpr int stage_bytes(int tokens) { return kLaneBytes + tokens * kTerms; }
struct SplitBarriers {
    uint64_t full[8], empty[8], done, sums;
    uint32_t tensor;
    int bad;
};
// (Kernels that hold tensor memory while they wait for another CTA must never share an SM with another such kernel whose CTA waits
// for tensor memory: this one's blocks take more than 44 KB, beside the 185 KB and more of kernels that have all 512 columns, and
// as many as fit an SM have at most 512 columns.)
__host__ __device__ constexpr int split_smem(int tokens) { return stages_of(tokens) * stage_bytes(tokens) + 1024 + 256 + tokens * 4; }

template <int TOKENS, class T>
__global__ void __launch_bounds__(kProductThreads, 1)
product_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, ProductArgs a, int tiles_n,
                     int kt, int* status) {
    constexpr int kStages = stages_of(TOKENS), kBytes = stage_bytes(TOKENS), kColumns = TOKENS < 32 ? 32 : TOKENS;
    extern __shared__ char raw[];
    char* stage = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    SplitBarriers* B = reinterpret_cast<SplitBarriers*>(stage + kStages * kBytes);
    float* token_scale = reinterpret_cast<float*>(reinterpret_cast<char*>(B) + 256);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const int tile = blockIdx.x / ranks;
    const int n0 = (tile % tiles_n) * kLanes;
    const long long m0 = static_cast<long long>(tile / tiles_n) * TOKENS;
    const int k_first = static_cast<int>(static_cast<long long>(kt) * rank / ranks);
    const int k_count = static_cast<int>(static_cast<long long>(kt) * (rank + 1) / ranks) - k_first;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&B->full[s], 1);
            mbar_init(&B->empty[s], 1);
        }
        mbar_init(&B->done, 1);
        mbar_init(&B->sums, 1);
        B->bad = 0;
        mbar_fence_init();
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_q);
    }
    const int early = a.w_early ? (k_count < kStages ? k_count : kStages) : 0;
    auto load_weight = [&](int i, int slot) {
        mbar_expect_tx(&B->full[slot], kBytes);
        load_tile(stage + slot * kBytes, &map_w, &B->full[slot], (k_first + i) * kTerms, n0);
    };
    __syncwarp();
    if (warp == 0 && elected())
        for (int i = 0; i < early; ++i) load_weight(i, i);
    __syncwarp();
    stream_order_begin();  // (tensor memory is asked for behind it: whoever is in front has given theirs back)
    if (warp == 1) tensor_alloc<1>(&B->tensor, kColumns);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tensor = B->tensor;
    auto give_up = [&]() {
        B->bad = 1;
        atomicExch(status, static_cast<int>(kDeviceTimeout));
    };
    if (warp == 0) {
        if (elected()) {
            int i = 0;
            RingPlace<kStages> at;
            for (; i < k_count; ++i, at.next()) {
                if (i >= kStages && !mbar_wait_bounded(&B->empty[at.stage], at.parity ^ 1)) {
                    give_up();
                    break;
                }
                if (i >= early) load_weight(i, at.stage);
                load_tile(stage + at.stage * kBytes + kLaneBytes, &map_q, &B->full[at.stage], (k_first + i) * kTerms, static_cast<int>(m0));
            }
            for (int j = i < kStages ? 0 : i - kStages; j < i; ++j)  // (no copy is in flight when the block ends)
                if (!mbar_wait_bounded(&B->full[j % kStages], (j / kStages) & 1)) give_up();
        }
    } else if (warp == 1) {
        if (elected()) {
            bool fine = true;
            RingPlace<kStages> at;
            const uint64_t w0 = operand(stage);
            for (int i = 0; i < k_count; ++i, at.next()) {
                fine = mbar_wait_bounded(&B->full[at.stage], at.parity);
                if (!fine) break;
                tensor_fence_after();
                const uint64_t w = w0 + at.stage * (kBytes >> 4), q = w + (kLaneBytes >> 4);
#pragma unroll
                for (int k = 0; k < kTerms / 32; ++k)
                    multiply<1>(tensor, w + 2 * k, q + 2 * k, product_kind(kLanes, TOKENS), i > 0 || k > 0);
                arrive_when_done<1>(&B->empty[at.stage]);
            }
            arrive_when_done<1>(&B->done);
            if (!fine) give_up();
        }
    } else {
        for (int c = threadIdx.x - 64; c < TOKENS; c += 32 * kStoreWarps) token_scale[c] = m0 + c < a.M ? a.scale[m0 + c] : 0.0f;
        if (!mbar_wait_bounded(&B->done, 0)) give_up();
        tensor_fence_after();
    }
    __syncthreads();
    // (a warp reaches the lanes 32 (warp % 4) .. + 31; the two of a quarter take every other step of its columns)
    const int quarter = warp & 3, turn = (warp - 2) >> 2, n = n0 + quarter * 32 + lane;
    const bool stores = warp >= 2;
    float w_scale = 0.0f, bias = 0.0f;
    if (stores && n < a.N) {
        w_scale = a.w_scale[n];
        bias = a.bias ? a.bias[n] : 0.0f;
    }
    T* out = static_cast<T*>(a.out);
    if (TOKENS == 256 || ranks == 1) {  // (256 tokens: there is no room for twice their sums)
        if (stores && !B->bad) {
            const int columns = a.M - m0 < TOKENS ? static_cast<int>(a.M - m0) : TOKENS;
            T* to = out + (m0 + 16 * turn) * a.N + n;
#pragma unroll 1
            for (int c = 16 * turn; c < columns; c += 32, to += 32LL * a.N) {
                int v[16];
                __syncwarp();
                tensor_load16(tensor + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
                tensor_load_wait(v);
                store16(a, v, token_scale + c, w_scale, bias, columns - c, n < a.N, to);
            }
        }
    } else {
        // Rank r gets the columns from first_of(r) on of every other rank's sums, [rank][column][128], behind its own sums where the
        // stages were.  As bulk copies: a thread's loads from another CTA wait a microsecond each, and its stores there, 4 bytes a
        // lane, took 65 clocks per column (512 tokens, 5120 -> 2048 in two shares: 17.6 us with loads, 15.0 with stores).
        auto first_of = [&](uint32_t r) { return static_cast<int>(TOKENS * r / ranks); };
        int* own = reinterpret_cast<int*>(stage);
        int* others = own + TOKENS * kLanes;
        const int first = first_of(rank), count = first_of(rank + 1) - first;
        if (stores) {
#pragma unroll 1
            for (int c = 16 * turn; c < TOKENS; c += 32) {
                int v[16];
                __syncwarp();
                tensor_load16(tensor + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
                tensor_load_wait(v);
#pragma unroll
                for (int j = 0; j < 16; ++j) own[(c + j) * kLanes + quarter * 32 + lane] = v[j];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the copies read them)
        } else if (threadIdx.x == 0) {
            mbar_expect_tx(&B->sums, (ranks - 1) * count * kLanes * 4);
        }
        __syncwarp();
        cluster_barrier();  // all products of all ranks have read what was there
        if (warp == 0) {
            if (elected())
                for (uint32_t r = 0; r < ranks; ++r)
                    if (r != rank) {
                        const int f = first_of(r), n_columns = first_of(r + 1) - f;
                        copy_to_cta(in_cta(others + (rank < r ? rank : rank - 1) * n_columns * kLanes, r), own + f * kLanes,
                                    n_columns * kLanes * 4, in_cta(&B->sums, r));
                    }
            __syncwarp();
        } else if (stores) {
            constexpr int kStep = 8;
            if (!mbar_wait_bounded(&B->sums, 0)) give_up();
            const int* mine = own + first * kLanes + quarter * 32 + lane;
            const int* theirs = others + quarter * 32 + lane;
            T* to = out + (m0 + first + kStep * turn) * a.N + n;
            const int columns = a.M - m0 - first < count ? static_cast<int>(a.M - m0 - first) : count;
#pragma unroll 1
            for (int c = kStep * turn; c < columns && !B->bad; c += 2 * kStep, to += 2LL * kStep * a.N) {
                int sum[kStep];
                float scale[kStep], value[kStep];
#pragma unroll
                for (int j = 0; j < kStep; ++j) {
                    sum[j] = c + j < count ? mine[(c + j) * kLanes] : 0;
                    scale[j] = c + j < count ? token_scale[first + c + j] : 0.0f;
                }
#pragma unroll 1
                for (uint32_t r = 0; r + 1 < ranks; ++r)
#pragma unroll
                    for (int j = 0; j < kStep; ++j)
                        if (c + j < count) sum[j] += theirs[(r * count + c + j) * kLanes];
                product_values(sum, scale, w_scale, bias, a.activation, value);
#pragma unroll
                for (int j = 0; j < kStep; ++j)
                    if (c + j < columns && n < a.N) to[static_cast<long long>(j) * a.N] = from_float<T>(value[j]);
            }
        }
        __syncwarp();
        cluster_barrier();  // this CTA's sums have arrived where they were sent
    }
    tensor_fence_before();
    __syncthreads();
    if (warp == 1) {
        tensor_fence_after();
        tensor_free<1>(tensor, kColumns);
    }
}

// ---- tiles of 256 outputs x 256 tokens for pairs of CTAs ----------------------------------------------------------------------
// For many tokens the products are what takes the time, and an SM cannot fetch as fast as 128 x 256 tiles would want it to: a
// pair's CTAs hold half of either operand each, 32 KB per CTA for 256 x 256 x 128 products.  A CTA keeps two tiles' sums in tensor
// memory, so that the stores of one run beside the products of the next.
constexpr int kPairStages = 6;
constexpr int kPairBytes = 2 * kLaneBytes;
constexpr int kPairTokens = 256;
struct PairBarriers {
    uint64_t full[kPairStages], empty[kPairStages], sums[2], taken[2];  // full, taken: those of the first CTA count
    uint32_t tensor;
    int bad;
};
__host__ __device__ constexpr int pair_smem() { return kPairStages * kPairBytes + 1024 + 256 + 2 * kPairTokens * 4; }

template <class T>
__global__ void __launch_bounds__(kProductThreads, 1)
product_pairs_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, ProductArgs a, int tiles_n,
                     int tiles, int kt, int* status) {
    extern __shared__ char raw[];
    char* stage = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    PairBarriers* B = reinterpret_cast<PairBarriers*>(stage + kPairStages * kPairBytes);
    float* scales = reinterpret_cast<float*>(reinterpret_cast<char*>(B) + 256);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(&B->full[s], 1);
            mbar_init(&B->empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&B->sums[s], 1);
            mbar_init(&B->taken[s], 2 * kStoreWarps);
        }
        B->bad = 0;
        mbar_fence_init();
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_q);
    }
    stream_order_begin();
    if (warp == 1) tensor_alloc<2>(&B->tensor, 512);
    tensor_fence_before();
    cluster_barrier();
    tensor_fence_after();
    const uint32_t tensor = B->tensor;
    auto give_up = [&]() {
        B->bad = 1;
        atomicExch(status, static_cast<int>(kDeviceTimeout));
    };
    if (warp == 0) {
        if (elected()) {
            long long i = 0;
            bool fine = true;
            RingPlace<kPairStages> at;
            for (int tile = pair; tile < tiles && fine; tile += pairs) {
                const int n = (tile % tiles_n) * 2 * kLanes + rank * kLanes, m = (tile / tiles_n) * kPairTokens + rank * kLanes;
                for (int k = 0; k < kt; ++k, ++i, at.next()) {
                    if (i >= kPairStages && !mbar_wait_bounded(&B->empty[at.stage], at.parity ^ 1)) {
                        fine = false;
                        give_up();
                        break;
                    }
                    const uint32_t full = in_cta(&B->full[at.stage], 0);
                    if (rank == 0) mbar_expect_tx(&B->full[at.stage], 2 * kPairBytes);
                    load_tile_of_pair(stage + at.stage * kPairBytes, &map_w, full, k * kTerms, n);
                    load_tile_of_pair(stage + at.stage * kPairBytes + kLaneBytes, &map_q, full, k * kTerms, m);
                }
            }
            // (nothing is in flight towards this CTA when it ends: neither its copies nor the pair's arrivals)
            // (an arrival there says that both CTAs' copies came and were read; without it, the copies are waited for as such)
            for (long long j = i < kPairStages ? 0 : i - kPairStages; j < i; ++j)
                if (!mbar_wait_bounded(&B->empty[j % kPairStages], (j / kPairStages) & 1)) {
                    give_up();
                    if (rank == 0) mbar_wait_bounded(&B->full[j % kPairStages], (j / kPairStages) & 1);
                }
        }
    } else if (warp == 1) {
        if (rank == 0 && elected()) {
            bool fine = true;
            int t = 0;
            RingPlace<kPairStages> at;
            const uint64_t w0 = operand(stage);
            for (int tile = pair; tile < tiles && fine; tile += pairs, ++t) {
                if (t >= 2 && !wait_bounded_cluster(&B->taken[t & 1], (t / 2 - 1) & 1)) {
                    fine = false;
                    break;
                }
                tensor_fence_after();
                for (int k = 0; k < kt; ++k, at.next()) {
                    fine = mbar_wait_bounded(&B->full[at.stage], at.parity);
                    if (!fine) break;
                    tensor_fence_after();
                    const uint64_t w = w0 + at.stage * (kPairBytes >> 4), q = w + (kLaneBytes >> 4);
#pragma unroll
                    for (int u = 0; u < kTerms / 32; ++u)
                        multiply<2>(tensor + (t & 1) * kPairTokens, w + 2 * u, q + 2 * u, product_kind(2 * kLanes, kPairTokens),
                                    k > 0 || u > 0);
                    arrive_when_done<2>(&B->empty[at.stage]);
                }
                if (fine) arrive_when_done<2>(&B->sums[t & 1]);
            }
            if (!fine) give_up();
        }
    } else {
        const int quarter = warp & 3, turn = (warp - 2) >> 2;
        T* out = static_cast<T*>(a.out);
        int t = 0;
        bool lost = false;  // the products of a tile did not come in time: this warp stores nothing more, but meets the others
        for (int tile = pair; tile < tiles; tile += pairs, ++t) {
            const int n = (tile % tiles_n) * 2 * kLanes + rank * kLanes + quarter * 32 + lane;
            const long long m0 = static_cast<long long>(tile / tiles_n) * kPairTokens;
            float w_scale = 0.0f, bias = 0.0f;
            if (n < a.N) {
                w_scale = a.w_scale[n];
                bias = a.bias ? a.bias[n] : 0.0f;
            }
            float* token_scale = scales + (t & 1) * kPairTokens;
            static_assert(kPairTokens == 32 * kStoreWarps, "a thread each");
            token_scale[threadIdx.x - 64] = m0 + threadIdx.x - 64 < a.M ? a.scale[m0 + threadIdx.x - 64] : 0.0f;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kStoreWarps) : "memory");  // (a tile later all have read the one before)
            // (one answer for the whole warp, whose loads and stores are common; and no warp leaves the loop, as the barrier above
            // counts all of them in every turn)
            if (lost) continue;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&B->sums[t & 1], (t / 2) & 1))) {
                give_up();
                lost = true;
                continue;
            }
            tensor_fence_after();
            const int columns = a.M - m0 < kPairTokens ? static_cast<int>(a.M - m0) : kPairTokens;
            T* to = out + (m0 + 16 * turn) * a.N + n;
#pragma unroll 1
            for (int c = 16 * turn; c < columns; c += 32, to += 32LL * a.N) {
                int v[16];
                __syncwarp();
                tensor_load16(tensor + (static_cast<uint32_t>(quarter * 32) << 16) + (t & 1) * kPairTokens + c, v);
                tensor_load_wait(v);
                store16(a, v, token_scale + c, w_scale, bias, columns - c, n < a.N, to);
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) arrive_remote(in_cta(&B->taken[t & 1], 0));
        }
    }
    __syncwarp();
    tensor_fence_before();
    cluster_barrier();
    if (warp == 1) {
        tensor_fence_after();
        tensor_free<2>(tensor, 512);
    }
}

}  // namespace
}  // namespace ldn
