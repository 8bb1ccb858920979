// The residual stream between two norms with rows in registers: forward one read of x, the residual and the gate and four sums over a row,
// backward one read of the five tensors that it takes and two rounds of sums, with the column sums carried in the threads that have those
// columns, from row to row.
//
// Bound by memory.  As in the layer norm's kernels, rows are under way into shared memory while others are summed, a block takes every
// gridDim-th row, so that its threads' columns and parameters stay (rows that start anywhere in 16 bytes: the grid is a multiple of
// eight, and rows that far apart start alike), and rows that are taken together share the barriers of their sums.  The scale and the first
// norm's parameters are two numbers per column, scale weight and scale bias.
//
// 16384 x 5120 bf16 with a gate of its shape: forward 180 us, 4.7 TB/s, backward 287, 4.7 (228 with the sums over rows left out: what the warps
// wait for); 8192 x 5120 float32 150 and 269; 524288 x 96 bf16 with a gate per row 146 and 236; 16383 x 4097 bf16, cut rows, 221 and 391;
// 8192 x 8192 bf16 215 and 376; 3457 x 8118 float32, shared by blocks, 229 and 345.
#pragma once
#include "ldn_sandwich.cuh"
#include "ldn_rows.cuh"
#include "ldn_tensor.cuh"

namespace ldn {
namespace {

template <Gate G>
constexpr int kForwardStreams = G == Gate::All ? 3 : 2;
template <Gate G, bool OF_Y>
constexpr int kBackwardStreams = (G == Gate::All ? 5 : 4) - (OF_Y ? 0 : 2);
constexpr int kMostRanks = 8;  // blocks of a cluster that share a row
// Threads of a block of rows (of 320, the compiler has as many registers for each as of 384)
__host__ __device__ constexpr int most_threads(int elements) { return elements <= 8 ? 640 : elements <= 16 ? 384 : 512; }
// Rows that a block, or each of its groups, takes at a time forward; backward one (524288 x 96 bf16 with a gate per row, 1 / 2 rows of a
// group: 172 / 146 us, backward 236 / 306; 1000000 x 17, cut rows: 107 / 111; 200000 x 40 f32: 45 / 43, four 49; groups of one lane, 4000000 x 8
// bf16 without a gate and with one per row, 2 / 4 rows: 57 / 63 and 142 / 138)
__host__ __device__ constexpr int rows_forward(int elements) { return elements > 16 ? 1 : 2; }

// scale weight and scale bias of a piece's columns (1 and 0 outside the row)
template <class T, bool SHIFT>
__device__ __forceinline__ void load_scaled(const SandwichParams& p, int c0, int C, float2 (&w)[kPiece<T> / 2], float2 (&b)[kPiece<T> / 2]) {
    float2 s[kPiece<T> / 2];
    load_params<T, SHIFT>(p.scale, p.wide, c0, C, 1.0f, s);
    load_params<T, SHIFT>(p.post_weight, p.wide, c0, C, 1.0f, w);
    load_params<T, SHIFT>(p.post_bias, p.wide, c0, C, 0.0f, b);
#pragma unroll
    for (int e = 0; e < kPiece<T> / 2; ++e) {
        w[e] = __fmul2_rn(w[e], s[e]);
        b[e] = __fmul2_rn(b[e], s[e]);
    }
}

// Numbers of the rows that a block takes next (statistics, a gate per row), in shared memory, some hundred rows at a time: fetched a turn ahead
// into registers, they were what the warps waited for (16384 x 5120 bf16 backward: 351 us with them, 277 without any).
constexpr int kNumberRows = 256;  // (times the rows that a group takes at a time: a turn's rows are there at least)
template <int N, int ROWS>
struct RowNumbers {
    float (*slots)[ROWS];
    int per_turn, turns;  // rows of a turn, turns of a batch
    __device__ __forceinline__ RowNumbers(float (*s)[ROWS], int rows_of_turn) : slots(s), per_turn(rows_of_turn), turns(ROWS / rows_of_turn) {}
    // load(k, row): number k of a row; row_of(i): the i-th row from this turn on, or rows and more where there is none
    template <class RowOf, class Load>
    __device__ __forceinline__ void at_turn(int turn, long long rows, RowOf row_of, Load load) {
        if (turn % turns) return;
        __syncthreads();
        for (int i = threadIdx.x; i < N * ROWS; i += blockDim.x) {
            const int k = i / ROWS, at = i % ROWS;
            const long long row = at < turns * per_turn ? row_of(at) : rows;
            slots[k][at] = row < rows ? load(k, row) : 0.0f;
        }
        __syncthreads();
    }
    // index: of a row in its turn
    __device__ __forceinline__ float of(int k, int turn, int index) const { return slots[k][turn % turns * per_turn + index]; }
};

// Sums over a block of rows held together, as RowSum has them, with the warps' sums read by all of a block's threads as whole pieces and
// added up by each (half the way of a second round of shuffles: the sums are what a block's warps wait for).  Sums over a
// group's lanes are RowSum's.
// The blocks of a cluster that share a row put their warps' sums into each other's memory and add up all of them.
enum class Share { Group, Block, Cluster };  // who has a row
template <Share W>
struct SumOf {
    int lanes;
    float* slots;  // [2][kSlots], zeros at first
    int turn, ranks, rank;
    static constexpr bool GROUP = W == Share::Group;
    static constexpr int kSlots = GROUP ? 4 : (W == Share::Cluster ? kMostRanks : 1) * 20 * 4;  // (warps of a row) x K, whole fours
    __device__ __forceinline__ void meet() {
        if constexpr (W == Share::Cluster) cluster_barrier();
        else __syncthreads();
    }
    __device__ __forceinline__ void begin() {
        if constexpr (!GROUP) {
            for (int i = threadIdx.x; i < 2 * kSlots; i += blockDim.x) slots[i] = 0.0f;
            meet();  // (and every block is there to be written to)
        }
    }
    template <int K, class End>
    __device__ __forceinline__ void operator()(float (&v)[K], End end) {
        if constexpr (GROUP) {
            RowSum{lanes, nullptr, 0}.over_group(v, [](float a, float b) { return a + b; }, end);
        } else {
            const int lane = threadIdx.x & 31;
            constexpr int kShare = 32 / K;  // lanes that end with the same number
            int half = 16;
#pragma unroll
            for (int n = K; n > 1; n /= 2, half /= 2) {
                const bool upper = lane & half;
#pragma unroll
                for (int i = 0; i < n / 2; ++i) {
                    const float send = upper ? v[i] : v[i + n / 2], keep = upper ? v[i + n / 2] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, half);
                }
            }
#pragma unroll
            for (int d = kShare / 2; d > 0; d /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
            float* s = slots + turn * kSlots;
            turn ^= 1;
            int warps = static_cast<int>(blockDim.x >> 5);
            const int at = static_cast<int>(threadIdx.x >> 5) * K + lane / kShare;
            if constexpr (W == Share::Cluster) {
                static_assert(kShare >= kMostRanks, "a lane for each block of a row");
                if (lane % kShare < ranks)
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(in_cta(s + rank * warps * K + at, lane % kShare)), "f"(v[0]) : "memory");
                warps *= ranks;
                __syncwarp();
            } else if (lane % kShare == 0) {
                s[at] = v[0];
            }
            meet();
            const int pieces = (warps * K + 3) / 4;
            const float4* from = reinterpret_cast<const float4*>(s);
            float4 a = from[0];
#pragma unroll 5
            for (int i = 1; i < pieces; ++i) {
                const float4 c = from[i];
                a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
            }
            if constexpr (K == 4) {
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            } else if constexpr (K == 2) {
                v[0] = a.x + a.z;
                v[1] = a.y + a.w;
            } else {
                v[0] = (a.x + a.y) + (a.z + a.w);
            }
#pragma unroll
            for (int i = 0; i < K; ++i) v[i] = end(v[i]);
        }
    }
};

// Blocks and rows under way: as many blocks per SM as registers allow, with what they may have of shared memory
struct RowShape {
    RowPlan p;
    int blocks, depth, ranks;  // blocks: of rows, each of so many of a cluster
    size_t smem;
};
// (sums' slots and rows' numbers)
template <Share W>
constexpr int kStaticBytes = (2 * SumOf<W>::kSlots + 5 * kNumberRows) * sizeof(float) + 256;
// Elements of a thread, threads of a block, and who has a row.  Whole blocks: 16 elements per thread of 16 bits (the instructions around an
// element count: 16384 x 5120 with 8 took 203 and 415 us), 8 of 32.  Longer rows: the blocks of a cluster; forward, where rows of 16 bits
// are whole, blocks with 32 elements per thread, which read their parameters again (8192 x 8192 bf16 221 us, in clusters 299; 4096 x 8192
// f32 313 and 201; backward 747, with the column sums in a kernel of their own, and 381).
bool plan_row(int C, int size, bool shift, bool forward, RowPlan* p, Share* who, int* ranks) {
    const int piece = 16 / size, elements = size == 4 ? 8 : 16, most = most_threads(elements);
    *ranks = 1;
    *who = Share::Block;
    if (plan_elements(C, size, shift, false, p) && p->group) {
        *who = Share::Group;
        return true;
    }
    if (plan_rows(C, piece, shift, elements / piece, most, p)) return true;
    if (forward && size == 2 && !shift && plan_rows(C, piece, shift, 32 / piece, most_threads(32), p)) return true;
    if (!plan_rows(C, piece, shift, elements / piece, kMostRanks * most, p)) return false;
    *who = Share::Cluster;
    *ranks = (p->lanes + most - 1) / most;
    p->threads = (p->lanes / 32 + *ranks - 1) / *ranks * 32;
    p->lanes = *ranks * p->threads;
    return true;
}
// What is on an SM: `per_sm` blocks that its registers hold, or fewer, so that rows are under way behind those that are worked on.
// extra, fixed: bytes of a block beside its rows
bool fill(const RowPlan& p, int R, int streams, long long extra, int fixed, const DeviceCtx* ctx, int* per_sm, int* depth) {
    const long long row_bytes = static_cast<long long>(R) * streams * p.items * p.threads * 16;
    auto room = [&] { return ctx->max_smem_optin / *per_sm - 1024 - fixed - extra; };
    *depth = ring_depth(row_bytes, room());
    while (*depth < 2 && *per_sm > 1) {
        --*per_sm;
        *depth = ring_depth(row_bytes, room());
    }
    return *depth >= 1;
}
// resident: blocks of rows (or clusters of them) that the device holds at a time
bool shape_of(const RowPlan& p, long long rows, int R, int streams, long long extra, int ranks, long long resident, int depth, RowShape* s) {
    s->p = p;
    s->ranks = ranks;
    s->depth = depth;
    const long long needed = (rows + p.rows_per_block() - 1) / p.rows_per_block();
    long long blocks = resident;
    if (p.shift && !p.group) {
        if (blocks < 8 && blocks < needed) return false;
        if (blocks >= 8) blocks = blocks / 8 * 8;
    }
    if (needed < blocks) blocks = needed;  // (a block has one row at most, then, and it does not matter how far they are apart)
    const long long turns = (needed + R * blocks - 1) / (R * blocks);
    if (turns < s->depth) s->depth = static_cast<int>(turns);
    s->blocks = static_cast<int>(blocks);
    s->smem = static_cast<size_t>(s->depth) * R * streams * p.items * p.threads * 16 + extra;
    return true;
}
// Calls f with a variant's numbers.
template <class T, bool FORWARD, class F>
int with_items(const RowPlan& p, Share who, F f) {
    constexpr int k8 = 8 / kPiece<T>, k16 = 16 / kPiece<T>, kBlock = sizeof(T) == 4 ? k8 : k16;
    using std::integral_constant;
    auto go = [&](auto items, auto share) { return p.shift ? f(items, share, std::true_type()) : f(items, share, std::false_type()); };
    constexpr auto group = integral_constant<Share, Share::Group>();
    constexpr auto block = integral_constant<Share, Share::Block>();
    if (who == Share::Group) return p.items == k8 ? go(integral_constant<int, k8>(), group) : go(integral_constant<int, k16>(), group);
    if (who == Share::Cluster) return go(integral_constant<int, kBlock>(), integral_constant<Share, Share::Cluster>());
    if constexpr (FORWARD && sizeof(T) == 2)
        if (p.items == 32 / kPiece<T>) return f(integral_constant<int, 32 / kPiece<T>>(), block, std::false_type());
    return go(integral_constant<int, kBlock>(), block);
}
template <class F>
int with_gate(Gate gate, F f) {
    switch (gate) {
        case Gate::None: return f(std::integral_constant<Gate, Gate::None>());
        case Gate::Row: return f(std::integral_constant<Gate, Gate::Row>());
        default: return f(std::integral_constant<Gate, Gate::All>());
    }
}
// The blocks of rows (or clusters of them) that the device holds at a time, and how many rows each has under way; false: not one
template <auto KERNEL, Share W>
bool resident_rows(const RowPlan& p, int R, int streams, long long extra, int ranks, const DeviceCtx* ctx, long long* resident, int* depth) {
    static OncePerDevice once;
    if (once([&] { return allow_smem(KERNEL, ctx->max_smem_optin - kStaticBytes<W>); }) != kOk) return false;
    static std::atomic<int> of_sm[64][33], of_device[64][33][kMostRanks + 1];
    auto asked = [](std::atomic<int>& known, auto ask) {
        int count = known.load(std::memory_order_acquire);
        if (count > 0) return count;
        if (ask(&count) != cudaSuccess || count < 1) {
            cudaGetLastError();
            count = 1;
        }
        known.store(count, std::memory_order_release);
        return count;
    };
    int per_sm = asked(of_sm[ctx->device][p.threads / 32],
                       [&](int* n) { return cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, KERNEL, p.threads, 0); });
    if (!fill(p, R, streams, extra, kStaticBytes<W>, ctx, &per_sm, depth)) return false;
    *resident = static_cast<long long>(per_sm) * ctx->sm_count;
    if (ranks > 1)
        *resident = asked(of_device[ctx->device][p.threads / 32][ranks], [&](int* n) {
            cudaLaunchAttribute attr[1] = {};
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = ranks;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(ctx->sm_count * per_sm / ranks * ranks);
            cfg.blockDim = dim3(p.threads);
            cfg.dynamicSmemBytes = static_cast<size_t>(*depth) * R * streams * p.items * p.threads * 16 + extra;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            return cudaOccupancyMaxActiveClusters(n, KERNEL, &cfg);
        });
    return true;
}

}  // namespace
}  // namespace ldn
