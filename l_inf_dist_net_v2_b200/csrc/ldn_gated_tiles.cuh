// The gated projection's products on the tensor cores: tcgen05.mma of 16-bit numbers, operands by TMA, 32-bit sums in tensor memory.
//
// Pairs of CTAs take tiles of 256 x 256 sums, a CTA 128 rows of them and half of either operand's loads.  Forward, the columns of a tile
// are 128 of the gate and the same 128 of the other projection (each CTA of a pair loads one of the two), so that a thread has both sums
// of an output and only the product leaves.  Operands are read as they lie in memory: for dx the weights, and for the weights' gradients
// both operands, have the terms as their rows, which the instruction takes as well (`across`).
//
// 32-bit operands are the sums of three bfloat16 images, 24 bits, and the six products of images down to 2^-18 are taken (what is left
// out is 2^-24 of a term or less): at the rate of 16-bit products a sixth, four times that of the 32-bit pipe.  The accumulator drops
// bits towards zero, 7e-8 of it per instruction on average, so sums stay in it for 256 terms at a time, small images first, and
// are added up in registers.  Sums of 16-bit products stay in it for 16384 terms (positive ones come 1e-4 too small at most, a fifth of what
// float16 rounds to); longer ones leave it after every 4096 (LONG): of 262144 terms they came 1.1e-3 too small, now 4e-5 (gradients of 2048 x
// 2048 weights in float16: 4.67 and 4.83 ms).
//
// What does not fill all pairs at the end is shared out among them in equal ranges of terms; a second kernel adds up the parts, in order.
//
// Bound by the tensor pipe where there are many rows: 16384, 5120 -> 5120 bf16, 1.72 TFLOP each way, 1.09 ms forward with both projections
// kept, 1.09 for dx, 1.09 for the weights' gradients (1.58 PFLOP/s; the library's product 1.63 in a burst).  512, 5120 -> 2048 float32, six
// products: 92, 89 and 93 us (1.40 PFLOP/s).  By start, fill, drain and the parts where there are few: 9 to 128 rows of 5120 -> 5120 29 to 39 us,
// of which the weights' bytes are 16.
#pragma once
#include "ldn_gated.cuh"
#include "ldn_tensor.cuh"

namespace ldn {
namespace {

constexpr int kSide = 256;           // of a tile
constexpr int kStepTerms = 64;       // 128 bytes of a row
constexpr int kHalfBytes = 128 * kStepTerms * 2;  // a CTA's share of an operand, per step
constexpr int kStepBytes = 2 * kHalfBytes;
constexpr int kStages = 6;
constexpr int kGroup = 8;            // rows of tiles that are walked through together, so that their operands are in L2
template <class T>
constexpr bool kParted = sizeof(T) == 4;
template <class T>
constexpr int kParts = kParted<T> ? 3 : 1;
// steps of a unit: of what is shared out, and at 32 bits of what stays in the accumulator (512 x 5120 -> 2048 in float32 with gradients,
// 2 / 4 / 8 steps: 381 / 374 / 382 us)
template <class T, bool LONG>
constexpr int kUnitSteps = kParted<T> ? 4 : LONG ? 64 : 1;
constexpr int kMostTerms = 16384;  // of 16 bits that stay in the accumulator
// the products of images, smallest first
__device__ __forceinline__ int part_of_a(int pass) { return (0x001102 >> 4 * pass) & 15; }
__device__ __forceinline__ int part_of_b(int pass) { return (0x010120 >> 4 * pass) & 15; }

struct TileBarriers {
    uint64_t full[kStages], empty[kStages], sums[2], taken[2];  // full, taken: those of the first CTA count
    uint32_t tensor;
};
constexpr int kTileSmem = kStages * kStepBytes + 1024 + 256;

template <class T>
__device__ __forceinline__ void multiply_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(kind), "r"(static_cast<uint32_t>(add))
                 : "memory");
}
// Operand whose rows are the terms: blocks of 64 columns (128 bytes, swizzled) x 64 terms, eight terms 1024 bytes apart; 16 terms further is
// 2048 bytes more
__device__ __forceinline__ uint64_t operand_across(const void* p) {
    return static_cast<uint64_t>((smem_u32(p) & 0x3ffffu) >> 4) | (static_cast<uint64_t>(kHalfBytes / 2 / 16) << 16) | (64ull << 32) |
           (1ull << 46) | (2ull << 61);
}
// 16-bit x 16-bit -> 32-bit sums of 256 x 256; across: the terms are the operand's rows
template <class T>
__host__ __device__ constexpr uint32_t kind_of(bool a_across, bool b_across) {
    return (1u << 4) | (std::is_same_v<T, __half> ? 0u : (1u << 7) | (1u << 10)) | (a_across ? 1u << 15 : 0u) | (b_across ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(kSide >> 3) << 17) | (static_cast<uint32_t>(kSide >> 4) << 24);
}
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint32_t bar, int inner, int row, int image) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(inner), "r"(row), "r"(image)
        : "memory");
}

// What a pair of CTAs takes: whole tiles in turn, then its range of the units of the others.
__host__ __device__ __forceinline__ long long range_begin(const TileArgs& a, int pair) {
    const long long all = static_cast<long long>(a.tiles - a.whole) * a.units;
    if (all < (1 << 24)) return static_cast<unsigned>(all) * static_cast<unsigned>(pair) / static_cast<unsigned>(a.pairs);  // (129 pairs at most)
    return all * pair / a.pairs;
}
struct Segments {
    int next_whole, tile, first, last, slot, later;
    long long at, end;
    bool part;  // of a tile, for the slot
    __device__ __forceinline__ Segments(const TileArgs& a, int pair)
        : next_whole(pair), slot(-1), later(2 * pair), at(range_begin(a, pair)), end(range_begin(a, pair + 1)), part(false) {}
    __device__ __forceinline__ bool next(const TileArgs& a) {
        if (next_whole < a.whole) {
            tile = next_whole;
            first = 0;
            last = a.units;
            next_whole += a.pairs;
            return true;
        }
        if (at >= end) return false;
        const int i = static_cast<int>(at / a.units);
        tile = a.whole + i;
        first = static_cast<int>(at - static_cast<long long>(i) * a.units);
        last = end - at < a.units - first ? first + static_cast<int>(end - at) : a.units;
        at += last - first;
        part = first > 0 || last < a.units;
        slot = later;  // (the first of a range has one, the last the other)
        later |= 1;
        return true;
    }
};
struct Place {
    int m, n;  // in tiles
};
__device__ __forceinline__ Place place_of(const TileArgs& a, int tile, int all_m) {
    const int per_group = kGroup * a.tiles_n, group = tile / per_group, r = tile - group * per_group;
    const int left = all_m - group * kGroup, high = left < kGroup ? left : kGroup;
    return {group * kGroup + r % high, r / high};
}

// 8 x 32 bits at a multiple of 32 bytes
__device__ __forceinline__ void store_32_bytes(void* to, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
template <class T>
__device__ __forceinline__ uint32_t two_of(float a, float b) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// N neighbouring values of which `columns` are there
template <class T, int N>
__device__ __forceinline__ void store_run(T* to, const float (&v)[N], int columns) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(to);
    if (columns >= N && (at & 31u) == 0 && N * sizeof(T) >= 32) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i + 8 <= N; i += 8) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[i + j]);
                store_32_bytes(to + i, w);
            }
        } else {
#pragma unroll
            for (int i = 0; i + 16 <= N; i += 16) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = two_of<T>(v[i + 2 * j], v[i + 2 * j + 1]);
                store_32_bytes(to + i, w);
            }
        }
    } else if (sizeof(T) == 4 && columns >= N && (at & 15u) == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(to + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else if (sizeof(T) == 2 && columns >= N && (at & 3u) == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) reinterpret_cast<uint32_t*>(to)[i / 2] = two_of<T>(v[i], v[i + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < columns) to[j] = from_float<T>(v[j]);
    }
}
// What follows the sums of N neighbouring columns of a row, from `n` on; forward: v0 the gate's, v1 the other projection's
template <class T, GatedForm F, int N>
__device__ __forceinline__ void finish(const TileArgs& a, int which, long long m, int n, float (&v0)[N], float (&v1)[N]) {
    const int columns = a.N - n;
    if (columns <= 0) return;
    if constexpr (F == GatedForm::Forward) {
        if (a.b_gate) {
#pragma unroll
            for (int j = 0; j < N; ++j) v0[j] += j < columns ? param_at<T>(a.b_gate, a.wide, n + j) : 0.0f;
        }
        if (a.b_up) {
#pragma unroll
            for (int j = 0; j < N; ++j) v1[j] += j < columns ? param_at<T>(a.b_up, a.wide, n + j) : 0.0f;
        }
        if (a.out1) {  // (rows of these are a whole number of runs)
            store_run<float, N>(static_cast<float*>(a.out1) + m * a.pitch_saved + n, v0, N);
            store_run<float, N>(static_cast<float*>(a.out2) + m * a.pitch_saved + n, v1, N);
        }
        activate(v0, a.activation);
#pragma unroll
        for (int j = 0; j < N; ++j) v0[j] *= v1[j];
        store_run<T, N>(static_cast<T*>(a.out0) + m * a.pitch + n, v0, columns);
    } else {
        store_run<T, N>(static_cast<T*>(F == GatedForm::GradWeights && which ? a.out1 : a.out0) + m * a.pitch + n, v0, columns);
    }
}

template <class T, GatedForm F, bool LONG>
__global__ void __launch_bounds__(kProductThreads, 1)
gated_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b0,
                   const __grid_constant__ CUtensorMap map_b1, const __grid_constant__ TileArgs a) {
    constexpr bool kGated = F == GatedForm::Forward, kAcrossA = F == GatedForm::GradWeights, kAcrossB = !kGated;
    constexpr bool kDrained = kParted<T> || LONG;  // sums leave the accumulator after every unit
    constexpr int kPasses = kParted<T> ? 6 : 1, kAheadA = kAcrossA ? 128 : 2, kAheadB = kAcrossB ? 128 : 2;
    constexpr uint32_t kKind = kind_of<T>(kAcrossA, kAcrossB);
    extern __shared__ char raw[];
    char* stage = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    TileBarriers* B = reinterpret_cast<TileBarriers*>(stage + kStages * kStepBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, all_m = F == GatedForm::GradWeights ? 2 * a.tiles_m : a.tiles_m;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&B->full[s], 1);
            mbar_init(&B->empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&B->sums[s], 1);
            mbar_init(&B->taken[s], 2 * kStoreWarps);
        }
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b0);
        tma_prefetch_desc(&map_b1);
    }
    stream_order_begin();
    if (warp == 1) tensor_alloc<2>(&B->tensor, 512);
    tensor_fence_before();
    cluster_barrier();
    tensor_fence_after();
    const uint32_t tensor = B->tensor;
    auto give_up = [&]() { atomicExch(a.status, static_cast<int>(kDeviceTimeout)); };
    // steps of a unit on its side (the two sides: dg with the gate's weights, du with the other's)
    auto steps_of = [&](int unit) {
        const int left = a.side_steps - (unit < a.side_units ? unit : unit - a.side_units) * kUnitSteps<T, LONG>;
        return left < kUnitSteps<T, LONG> ? left : kUnitSteps<T, LONG>;
    };
    Segments seg(a, pair);
    if (warp == 0) {
        if (elected()) {
            long long i = 0;
            bool fine = true;
            RingPlace<kStages> at;
            while (fine && seg.next(a)) {
                const Place p = place_of(a, seg.tile, all_m);
                const int which = F == GatedForm::GradWeights && p.m >= a.tiles_m;
                const int m = (which ? p.m - a.tiles_m : p.m) * kSide + rank * 128;
                const int n = kGated ? p.n * 128 : p.n * kSide + rank * 128;
                for (int u = seg.first; u < seg.last && fine; ++u) {
                    const int side = u >= a.side_units, steps = steps_of(u);
                    const int term0 = (u - (side ? a.side_units : 0)) * kUnitSteps<T, LONG> * kStepTerms;
                    const CUtensorMap* map_b = (kGated ? rank : side) ? &map_b1 : &map_b0;
                    const int first_image = (F == GatedForm::GradRows ? side : which) * kParts<T>;
#pragma unroll 1
                    for (int pass = 0; pass < kPasses && fine; ++pass) {
                        const int image_a = first_image + (kPasses > 1 ? part_of_a(pass) : 0), image_b = kPasses > 1 ? part_of_b(pass) : 0;
                        for (int k = 0; k < steps; ++k, ++i, at.next()) {
                            if (i >= kStages && !mbar_wait_bounded(&B->empty[at.stage], at.parity ^ 1)) {
                                fine = false;
                                give_up();
                                break;
                            }
                            const uint32_t full = in_cta(&B->full[at.stage], 0);
                            if (rank == 0) mbar_expect_tx(&B->full[at.stage], 2 * kStepBytes);
                            char *to_a = stage + at.stage * kStepBytes, *to_b = to_a + kHalfBytes;
                            const int term = term0 + k * kStepTerms;
                            if constexpr (kAcrossA) {
                                load_box(to_a, &map_a, full, m, term, image_a);
                                load_box(to_a + kHalfBytes / 2, &map_a, full, m + 64, term, image_a);
                            } else {
                                load_box(to_a, &map_a, full, term, m, image_a);
                            }
                            if constexpr (kAcrossB) {
                                load_box(to_b, map_b, full, n, term, image_b);
                                load_box(to_b + kHalfBytes / 2, map_b, full, n + 64, term, image_b);
                            } else {
                                load_box(to_b, map_b, full, term, n, image_b);
                            }
                        }
                    }
                }
            }
            // (nothing is in flight towards this CTA when it ends: an arrival says that both CTAs' copies came and were read; without it,
            // the copies are waited for as such)
            for (long long j = i < kStages ? 0 : i - kStages; j < i; ++j)
                if (!mbar_wait_bounded(&B->empty[j % kStages], (j / kStages) & 1)) {
                    give_up();
                    if (rank == 0) mbar_wait_bounded(&B->full[j % kStages], (j / kStages) & 1);
                }
        }
    } else if (warp == 1) {
        if (rank == 0 && elected()) {
            bool fine = true;
            int batch = 0;  // sums that leave together: a segment's, or a unit's
            RingPlace<kStages> at;
            const uint64_t a0 = kAcrossA ? operand_across(stage) : operand(stage);
            const uint64_t b0 = kAcrossB ? operand_across(stage + kHalfBytes) : operand(stage + kHalfBytes);
            while (fine && seg.next(a)) {
                bool add = false;
                for (int u = seg.first; u < seg.last && fine; ++u) {
                    if (kDrained || u == seg.first) {
                        if (batch >= 2 && !wait_bounded_cluster(&B->taken[batch & 1], (batch / 2 - 1) & 1)) {
                            fine = false;
                            break;
                        }
                        tensor_fence_after();
                        add = false;
                    }
                    const int steps = steps_of(u) * kPasses;
                    for (int k = 0; k < steps; ++k, at.next()) {
                        fine = mbar_wait_bounded(&B->full[at.stage], at.parity);
                        if (!fine) break;
                        tensor_fence_after();
                        const uint64_t da = a0 + at.stage * (kStepBytes >> 4), db = b0 + at.stage * (kStepBytes >> 4);
#pragma unroll
                        for (int j = 0; j < kStepTerms / 16; ++j)
                            multiply_pair<T>(tensor + (batch & 1) * kSide, da + kAheadA * j, db + kAheadB * j, kKind, add || j > 0);
                        add = true;
                        arrive_when_done<2>(&B->empty[at.stage]);
                    }
                    if (fine && (kDrained || u == seg.last - 1)) {
                        arrive_when_done<2>(&B->sums[batch & 1]);
                        ++batch;
                    }
                }
            }
            if (!fine) give_up();
        }
    } else {
        // A warp reaches the lanes 32 (warp % 4) .. + 31; the two of a quarter have half of the columns each, in runs of 16.
        const int quarter = warp & 3, half = (warp - 2) >> 2, row = rank * 128 + quarter * 32 + lane;
        const uint32_t lanes = tensor + (static_cast<uint32_t>(quarter * 32) << 16);
        auto column = [&](int run) {  // of a tile's sums; forward: four runs of the gate, then the same of the other projection
            return kGated ? (run < 4 ? 0 : 64) + 64 * half + 16 * run : 128 * half + 16 * run;
        };
        int batch = 0;
        bool lost = false;
        auto wait = [&]() {
            if (__all_sync(0xffffffffu, mbar_wait_bounded(&B->sums[batch & 1], (batch / 2) & 1))) {
                tensor_fence_after();
                return true;
            }
            give_up();
            lost = true;
            return false;
        };
        auto taken = [&]() {
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) arrive_remote(in_cta(&B->taken[batch & 1], 0));
            ++batch;
        };
        while (!lost && seg.next(a)) {
            const Place p = place_of(a, seg.tile, all_m);
            const int which = F == GatedForm::GradWeights && p.m >= a.tiles_m;
            const long long m = static_cast<long long>(which ? p.m - a.tiles_m : p.m) * kSide + row;
            const int n = kGated ? p.n * 128 + 64 * half : p.n * kSide + 128 * half;  // of this warp's first run
            float* part = a.partials + (static_cast<size_t>(seg.slot) * kSide + row) * kSide;
            if constexpr (kDrained) {
                float acc[8][16];
#pragma unroll
                for (int r = 0; r < 8; ++r)
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[r][j] = 0.0f;
                for (int u = seg.first; u < seg.last; ++u) {
                    if (!wait()) break;
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        int v[16];
                        __syncwarp();
                        tensor_load16(lanes + (batch & 1) * kSide + column(r), v);
                        tensor_load_wait(v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[r][j] += __int_as_float(v[j]);
                    }
                    taken();
                }
                if (lost || m >= a.M) continue;
                if (seg.part) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) store_run<float, 16>(part + column(r), acc[r], 16);
                } else if constexpr (kGated) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) finish<T, F, 16>(a, which, m, n + 16 * r, acc[r], acc[r + 4]);
                } else {
#pragma unroll
                    for (int r = 0; r < 8; ++r) finish<T, F, 16>(a, which, m, n + 16 * r, acc[r], acc[r]);
                }
            } else {
                if (!wait()) break;
                constexpr int kRuns = kGated ? 4 : 8;
#pragma unroll 1
                for (int r = 0; r < kRuns; ++r) {
                    int v[16], w[16];
                    float f[16], h[16];
                    __syncwarp();
                    tensor_load16(lanes + (batch & 1) * kSide + column(r), v);
                    if constexpr (kGated) tensor_load16(lanes + (batch & 1) * kSide + column(r + 4), w);
                    tensor_load_wait(v);
                    if constexpr (kGated) tensor_load_wait(w);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        f[j] = __int_as_float(v[j]);
                        h[j] = kGated ? __int_as_float(w[j]) : 0.0f;
                    }
                    if (m < a.M) {
                        if (seg.part) {
                            store_run<float, 16>(part + column(r), f, 16);
                            if constexpr (kGated) store_run<float, 16>(part + column(r + 4), h, 16);
                        } else {
                            finish<T, F, 16>(a, which, m, n + 16 * r, f, h);
                        }
                    }
                }
                taken();
            }
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

// The parts of a tile that several pairs share, added up in the order of their terms; a block has four rows of a tile, a thread four columns.
// Which pairs have a part is found by a thread each, and four parts are under way at a time (found and loaded one after the other, 15 parts
// of 64 rows took 29 us; four at a time 11, eight 14).
constexpr int kFixRows = 4, kFixAhead = 4, kMostPairs = 128;
template <GatedForm F>
constexpr int kFixRuns = F == GatedForm::Forward ? 32 : 64;  // of four columns
template <class T, GatedForm F>
__global__ void __launch_bounds__(kFixRows * kFixRuns<F>) gated_parts_kernel(const __grid_constant__ TileArgs a) {
    stream_order_begin();
    constexpr bool kGated = F == GatedForm::Forward;
    __shared__ int slots[kMostPairs], first, last, alone;
    const int i = blockIdx.x, all_m = F == GatedForm::GradWeights ? 2 * a.tiles_m : a.tiles_m;
    const long long begin = static_cast<long long>(i) * a.units, end = begin + a.units;
    if (threadIdx.x == 0) {
        first = kMostPairs;
        last = alone = 0;
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < a.pairs) {
        const int q = threadIdx.x;
        const long long b = range_begin(a, q), e = range_begin(a, q + 1);
        const bool there = b < e && b < end && e > begin;
        slots[q] = there ? 2 * q + (b < begin) : -1;
        if (there) {
            atomicMin(&first, q);
            atomicMax(&last, q);
            if (b <= begin && e >= end) alone = 1;
        }
    }
    __syncthreads();
    if (alone) return;  // (one pair has all of the tile, and has stored it)
    const Place p = place_of(a, a.whole + i, all_m);
    const int which = F == GatedForm::GradWeights && p.m >= a.tiles_m;
    const int row = blockIdx.y * kFixRows + threadIdx.x / kFixRuns<F>, run = threadIdx.x % kFixRuns<F>;
    const long long m = static_cast<long long>(which ? p.m - a.tiles_m : p.m) * kSide + row;
    const int n = kGated ? p.n * 128 + 4 * run : p.n * kSide + 4 * run;
    if (m >= a.M || n >= a.N) return;
    const float* from = a.partials + static_cast<size_t>(row) * kSide + 4 * run;
    float v0[4] = {}, v1[4] = {};
    for (int q0 = first; q0 <= last; q0 += kFixAhead) {
        float4 s[kFixAhead], t[kFixAhead];
#pragma unroll
        for (int j = 0; j < kFixAhead; ++j) {
            const int slot = q0 + j <= last ? slots[q0 + j] : -1;
            s[j] = t[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (slot >= 0) {
                const float* f = from + static_cast<size_t>(slot) * kSide * kSide;
                s[j] = *reinterpret_cast<const float4*>(f);
                if constexpr (kGated) t[j] = *reinterpret_cast<const float4*>(f + 128);
            }
        }
#pragma unroll
        for (int j = 0; j < kFixAhead; ++j) {
            v0[0] += s[j].x; v0[1] += s[j].y; v0[2] += s[j].z; v0[3] += s[j].w;
            if constexpr (kGated) { v1[0] += t[j].x; v1[1] += t[j].y; v1[2] += t[j].z; v1[3] += t[j].w; }
        }
    }
    finish<T, F, 4>(a, which, m, n, v0, v1);
}

}  // namespace
}  // namespace ldn
