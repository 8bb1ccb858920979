// Layer norm's gradient with the row on the SM: one read of x and of the incoming gradients, both sums over a row at once, and the
// column sums for the weight and the bias carried in the threads that have those columns, from row to row.
//
// A block takes every gridDim-th row, so its threads' columns stay (rows that start anywhere in 16 bytes: the grid is a multiple of
// eight, and rows that far apart start alike).  Rows are under way into shared memory while others are summed, as in the forward
// pass, and are read there twice: in front of the sums and behind them.  Bound by memory: x, the incoming and the outgoing gradients
// once; joined, also by the latency of the dropout's words.  16384 x 5120 bf16: 97 us, 5.2 TB/s (50000 rows: 265 us, 5.8 TB/s; joined
// 589, 4.3; 16383 x 4097, cut rows: 132, 3.0; 8192 x 5120 f32: 91, 5.5).  Rows beyond 5120 take the parameters again for every row, one
// row at a time: 8192 x 8192 bf16 132 us, 3.0 TB/s.
#include "ldn_norm.cuh"
#include "ldn_rows.cuh"

namespace ldn {
namespace {

// Rows that a block takes at a time, so that their sums share their barriers
__host__ __device__ constexpr int rows_at_once(bool joined, int elements, bool group) {
    return group || elements > 16 ? 1 : elements > 8 || joined ? 2 : 4;
}
template <bool JOINED>
constexpr int kStreams = JOINED ? 3 : 2;

template <int N>
__device__ __forceinline__ float at_of(const float2 (&v)[N], int e) {
    return e % 2 ? v[e / 2].y : v[e / 2].x;
}

template <class T, bool JOINED, int ITEMS, bool GROUP, bool SHIFT>
__global__ void __launch_bounds__(GROUP ? kGroupThreads : threads_of(ITEMS * kPiece<T>), !GROUP && ITEMS * kPiece<T> == 16 ? 2 : 1) norm_grad_registers_kernel(NormGradArgs a, int lanes, int depth) {
    stream_order_begin();
    constexpr int V = kPiece<T>, S = kStreams<JOINED>, R = rows_at_once(JOINED, ITEMS * V, GROUP);
    constexpr bool kStatsCome = !GROUP && sizeof(T) == 2;
    constexpr bool kKeep = ITEMS * V <= 16;  // the columns' weights stay in registers, too
    __shared__ float slots[2 * RowSum::kSlots];
    extern __shared__ uint4 ring[];  // [depth][row][stream][item][thread], then [warp][depth][row][2] floats; at the end, groups: [warp][2][C] floats
    RowSum reduce{lanes, slots, 0};
    Generator gen;
    if constexpr (JOINED) gen = generator_of(a.drop);
    const int lane = GROUP ? threadIdx.x & (lanes - 1) : threadIdx.x;
    const int per_block = GROUP ? kGroupThreads / lanes : 1;
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    const long long mine = static_cast<long long>(blockIdx.x) * per_block + (GROUP ? threadIdx.x / lanes : 0);
    const float inv_C = 1.0f / a.C;
    // (the same for all rows of this thread)
    const int shift = SHIFT ? shift_of(static_cast<const T*>(a.x) + (mine < a.rows ? mine : 0) * a.pitch) : 0;
    auto column = [&](int i) { return (lane + i * lanes) * V - shift; };
    float2 sum_w[ITEMS][V / 2], sum_b[ITEMS][V / 2], w[ITEMS][V / 2];
    uint4 mask[ITEMS];
    int bytes[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) sum_w[i][e] = sum_b[i][e] = both(0.0f);
        mask[i] = mask_of<T, SHIFT>(column(i), a.C);
        bytes[i] = piece_bytes<T>(column(i), a.C);
        if constexpr (kKeep) load_params<T, SHIFT>(a.weight, a.wide, column(i), a.C, 1.0f, w[i]);
    }
    // this thread's rows, and where their pieces are: those to be fetched, and those to be made
    const int c0 = column(0), apart = lanes * V;
    int to_fetch = mine < a.rows ? static_cast<int>((a.rows - mine + step - 1) / step) : 0, to_make = to_fetch;
    Walk<const T> from_x(a.x, a.pitch, mine, step, c0), from_y(a.grad_y, a.C, mine, step, c0), from_h(a.grad_h, a.C, mine, step, c0);
    Walk<T> to_x(a.grad_x, a.C, mine, step, c0), to_h(a.grad_residual, a.C, mine, step, c0);
    long long row0 = mine, index = mine * a.C + c0;
    uint4* own = ring + threadIdx.x;
    auto slot_of = [&](int stage, int j, int stream, int i) { return own + (((stage * R + j) * S + stream) * ITEMS + i) * blockDim.x; };
    float* stats = reinterpret_cast<float*>(ring + static_cast<size_t>(depth) * R * S * ITEMS * blockDim.x) + (threadIdx.x >> 5) * depth * 2 * R;
    const float* from_stat = ((threadIdx.x & 1) ? a.rstd : a.mean) + mine + (threadIdx.x & 31) / 2 * step;
    auto fetch = [&](int stage) {
        if (kStatsCome) {
            const int k = threadIdx.x & 31;  // mean and 1 / deviation of row k / 2
            if (k < 2 * R && k / 2 < to_fetch) copy_async<4>(stats + stage * 2 * R + k, from_stat, 4);
            from_stat += R * step;
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (j < to_fetch) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    copy_piece<T, SHIFT>(slot_of(stage, j, 0, i), from_x.of(j, i * apart), column(i), bytes[i], a.x);
                    copy_piece<T, SHIFT>(slot_of(stage, j, 1, i), from_y.of(j, i * apart), column(i), bytes[i], a.grad_y);
                    if constexpr (JOINED)
                        if (a.grad_h) copy_piece<T, SHIFT>(slot_of(stage, j, 2, i), from_h.of(j, i * apart), column(i), bytes[i], a.grad_h);
                }
            }
        copies_commit();
        to_fetch -= R;
        from_x.on(R);
        from_y.on(R);
        if (JOINED) from_h.on(R);
    };
    for (int d = 0; d < depth * R * S; ++d)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (!bytes[i]) own[(d * ITEMS + i) * blockDim.x] = make_uint4(0u, 0u, 0u, 0u);
    for (int d = 0; d < depth; ++d) fetch(d);
    // The statistics of the next turn's rows: loaded when they were wanted, they were what 16-bit rows waited for most (16384 x 5120:
    // 119 us, 108 so).  Blocks of such have them come with the rows, a warp's first lanes for the warp; groups have registers for them;
    // 32-bit blocks, with more bytes to wait for, load them at once (8192 x 5120: 92 us, 97 the other way).
    float next_mean[R], next_rstd[R];
    auto fetch_stats = [&](long long row, int rows) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            next_mean[j] = j < rows ? a.mean[row + j * step] : 0.0f;
            next_rstd[j] = j < rows ? a.rstd[row + j * step] : 0.0f;
        }
    };
    if (GROUP) fetch_stats(row0, to_make);
    int stage = 0;
    // (a warp's groups take part in its shuffles whether they have a row or not: as many turns as the block's first has)
    const long long block_first = static_cast<long long>(blockIdx.x) * per_block;
    const int turns = block_first < a.rows ? static_cast<int>((a.rows - block_first + R * step - 1) / (R * step)) : 0;
    for (int turn = 0; turn < turns; ++turn) {
        auto live = [&](int j) { return j < to_make; };
        float mean[R], rstd[R], s[2 * R];
        if constexpr (!GROUP && !kStatsCome) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                mean[j] = live(j) ? a.mean[row0 + j * step] : 0.0f;
                rstd[j] = live(j) ? a.rstd[row0 + j * step] : 0.0f;
            }
        }
        copies_wait(depth);
        if constexpr (GROUP) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                mean[j] = next_mean[j];
                rstd[j] = next_rstd[j];
            }
            fetch_stats(row0 + R * step, to_make - R);
        } else if constexpr (kStatsCome) {
            __syncwarp();  // (the lane that copied them has waited)
#pragma unroll
            for (int j = 0; j < R; ++j) {
                mean[j] = live(j) ? stats[stage * 2 * R + 2 * j] : 0.0f;
                rstd[j] = live(j) ? stats[stage * 2 * R + 2 * j + 1] : 0.0f;
            }
            __syncwarp();
        }
        // (outside the row the gradient is 0, and x a number; where there is no row, all is 0)
        auto piece_of = [&](int j, int stream, int i) {
            uint4 raw = live(j) ? *slot_of(stage, j, stream, i) : make_uint4(0u, 0u, 0u, 0u);
            return SHIFT ? masked(raw, mask[i]) : raw;
        };
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                float2 vx[V / 2], vg[V / 2];
                unpack<T>(piece_of(j, 0, i), vx);
                unpack<T>(piece_of(j, 1, i), vg);
                if constexpr (!kKeep) load_params<T, SHIFT>(a.weight, a.wide, column(i), a.C, 1.0f, w[i]);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    // (what is summed is a (x - mean), with rstd behind the sum: outside the row the gradient is 0 and x - mean a
                    // number, but (0 - mean) rstd may be infinite.  Two orders of the products, for their registers: 50000 x 4096
                    // bf16 208 and 226 us, joined 507 and 505, cut rows of 4097 in f16 410 and 370)
                    const float2 d = __fadd2_rn(vx[e], both(-mean[j]));
                    sum_b[i][e] = __fadd2_rn(sum_b[i][e], vg[e]);
                    if constexpr (!SHIFT && !JOINED) {
                        const float2 p = __fmul2_rn(vg[e], w[i][e]);
                        s0 = __fadd2_rn(s0, p);
                        s1 = __ffma2_rn(p, d, s1);
                        sum_w[i][e] = __ffma2_rn(vg[e], __fmul2_rn(d, both(rstd[j])), sum_w[i][e]);
                    } else {
                        const float2 u = __fmul2_rn(vg[e], d);
                        sum_w[i][e] = __ffma2_rn(u, both(rstd[j]), sum_w[i][e]);
                        s0 = __ffma2_rn(vg[e], w[i][e], s0);
                        s1 = __ffma2_rn(u, w[i][e], s1);
                    }
                }
            }
            s[2 * j] = s0.x + s0.y;
            s[2 * j + 1] = s1.x + s1.y;
        }
        reduce.template sum<GROUP>(s, [&](float all) { return all * inv_C; });
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (!live(j)) continue;
            const float m1 = s[2 * j], m2 = s[2 * j + 1] * rstd[j] * rstd[j];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = column(i);
                float2 vx[V / 2], vg[V / 2];
                unpack<T>(piece_of(j, 0, i), vx);
                unpack<T>(piece_of(j, 1, i), vg);
                if constexpr (!kKeep) load_params<T, SHIFT>(a.weight, a.wide, c, a.C, 1.0f, w[i]);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 p = __ffma2_rn(vg[e], w[i][e], both(-m1));
                    vg[e] = __fmul2_rn(__ffma2_rn(__fadd2_rn(vx[e], both(-mean[j])), both(-m2), p), both(rstd[j]));
                }
                if constexpr (JOINED) {
                    if (a.grad_h) {
                        float2 vh[V / 2];
                        unpack<T>(piece_of(j, 2, i), vh);
#pragma unroll
                        for (int e = 0; e < V / 2; ++e) vg[e] = __fadd2_rn(vg[e], vh[e]);
                    }
                    if (a.grad_residual) store_piece<T, SHIFT>(to_h.of(j, i * apart), c, a.C, pack<T>(vg));
                    if (a.grad_x) drop_piece(a.drop, gen, index + j * step * a.C + i * apart, vg);  // (pieces start at multiples of four)
                }
                if (a.grad_x) store_piece<T, SHIFT>(to_x.of(j, i * apart), c, a.C, pack<T>(vg));
            }
        }
        fetch(stage);
        stage = stage + 1 == depth ? 0 : stage + 1;
        to_make -= R;
        row0 += R * step;
        to_x.on(R);
        if (JOINED) {
            to_h.on(R);
            index += R * step * a.C;
        }
    }
    if (!a.parts) return;
    float* part = a.parts + static_cast<long long>(blockIdx.x) * 2 * a.C;
    if constexpr (!GROUP) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = column(i);
            if constexpr (!SHIFT) {
                if (c >= a.C) continue;
#pragma unroll
                for (int e = 0; e < V / 2; e += 2) {
                    *reinterpret_cast<float4*>(part + c + 2 * e) = make_float4(sum_w[i][e].x, sum_w[i][e].y, sum_w[i][e + 1].x, sum_w[i][e + 1].y);
                    *reinterpret_cast<float4*>(part + a.C + c + 2 * e) =
                        make_float4(sum_b[i][e].x, sum_b[i][e].y, sum_b[i][e + 1].x, sum_b[i][e + 1].y);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (static_cast<unsigned>(c + e) < static_cast<unsigned>(a.C)) {
                        part[c + e] = at_of(sum_w[i], e);
                        part[a.C + c + e] = at_of(sum_b[i], e);
                    }
            }
        }
    } else {
        // a warp's groups add to its columns in turn, then the warps' are added up
        float* columns = reinterpret_cast<float*>(ring);
        copies_wait(1);
        __syncthreads();  // (all have read their rows)
        float* own = columns + (threadIdx.x >> 5) * 2 * a.C;
        const int turn = (threadIdx.x & 31) / lanes;
        for (int k = 0; k < 32 / lanes; ++k) {
            if (turn == k)
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const int c0 = (lane + i * lanes) * V - shift;
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(a.C)) {
                            own[c0 + e] = at_of(sum_w[i], e) + (k ? own[c0 + e] : 0.0f);
                            own[a.C + c0 + e] = at_of(sum_b[i], e) + (k ? own[a.C + c0 + e] : 0.0f);
                        }
                }
            __syncwarp();
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * a.C; c += kGroupThreads) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kGroupThreads / 32; ++w) s += columns[w * 2 * a.C + c];
            part[c] = s;
        }
    }
}

struct GradShape {
    RowPlan p;
    int blocks, depth;
    size_t smem;
};

bool plan_of(bool joined, const NormGradArgs& a, int type, const DeviceCtx* ctx, GradShape* s) {
    const int size = size_of(type);
    const bool aligned = on16(a.x) && on16(a.grad_y) && on16(a.grad_h) && on16(a.grad_x) && on16(a.grad_residual);
    const bool shift = rows_shift(size, a.C) || !on16(a.weight);
    RowPlan& p = s->p;
    if (!rows_match(size, a.C, a.pitch, aligned) ||
        !plan_elements(a.C, size, shift, joined, &p))
        return false;
    const int elements = p.items * (16 / size), R = rows_at_once(joined, elements, p.group);
    const long long row_bytes = static_cast<long long>(R) * (joined ? 3 : 2) * p.items * p.threads * 16, most_smem = ctx->max_smem_optin - 4096;
    // blocks per SM: up to 102 registers per thread, 128 with 32 elements, and rows under way behind those that are summed
    int per_sm = 65536 / (p.threads * (elements <= 16 ? 102 : 128));
    if (per_sm > 4) per_sm = 4;
    if (per_sm < 1) per_sm = 1;
    s->depth = ring_depth(row_bytes, most_smem / per_sm - 1024);
    while (s->depth < 2 && per_sm > 1) s->depth = ring_depth(row_bytes, most_smem / --per_sm - 1024);
    if (s->depth < 1) s->depth = 1;  // (rows of 16384 in 32 bits: 128 KB, joined 192 KB)
    const long long needed = (a.rows + p.rows_per_block() - 1) / p.rows_per_block();
    long long blocks = static_cast<long long>(per_sm) * ctx->sm_count;
    if (p.shift && !p.group) blocks = blocks / 8 * 8;
    if (needed < blocks) blocks = needed;
    const long long turns = (needed + R * blocks - 1) / (R * blocks);
    if (turns < s->depth) s->depth = static_cast<int>(turns);
    s->blocks = static_cast<int>(blocks);
    s->smem = static_cast<size_t>(s->depth) * (row_bytes + (p.threads / 32) * R * 2 * sizeof(float));
    const size_t columns = p.group ? static_cast<size_t>(kGroupThreads / 32) * 2 * a.C * sizeof(float) : 0;
    if (s->smem < columns) s->smem = columns;
    return true;
}

template <class T, bool JOINED, int ITEMS, bool GROUP, bool SHIFT>
int run(const NormGradArgs& a, const GradShape& s, const DeviceCtx* ctx, cudaStream_t st) {
    constexpr auto kernel = norm_grad_registers_kernel<T, JOINED, ITEMS, GROUP, SHIFT>;
    static OncePerDevice once;
    const int r = once([&] { return allow_smem(kernel, ctx->max_smem_optin - 2560); });
    if (r != kOk) return r;
    return launch_after(kernel, s.blocks, s.p.threads, s.smem, st, a, s.p.lanes, s.depth);
}
template <class T, bool JOINED>
int run(const NormGradArgs& a, const GradShape& s, const DeviceCtx* ctx, cudaStream_t st) {
    constexpr int k8 = 8 / kPiece<T>, k16 = 16 / kPiece<T>, k32 = 32 / kPiece<T>;
    constexpr int kBlock = JOINED || sizeof(T) == 4 ? k8 : k16;  // (as plan_elements has it)
    const RowPlan& p = s.p;
    if (p.group && p.items == k8)
        return p.shift ? run<T, JOINED, k8, true, true>(a, s, ctx, st) : run<T, JOINED, k8, true, false>(a, s, ctx, st);
    if (p.group) return p.shift ? run<T, JOINED, k16, true, true>(a, s, ctx, st) : run<T, JOINED, k16, true, false>(a, s, ctx, st);
    if (p.items == kBlock)
        return p.shift ? run<T, JOINED, kBlock, false, true>(a, s, ctx, st) : run<T, JOINED, kBlock, false, false>(a, s, ctx, st);
    return p.shift ? run<T, JOINED, k32, false, true>(a, s, ctx, st) : run<T, JOINED, k32, false, false>(a, s, ctx, st);
}

}  // namespace

bool norm_grad_in_registers(bool joined, const NormGradArgs& a, int type, const DeviceCtx* ctx, int* blocks) {
    GradShape s;
    if (!plan_of(joined, a, type, ctx, &s)) return false;
    *blocks = s.blocks;
    return true;
}

int launch_norm_grad_in_registers(bool joined, const NormGradArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st) {
    GradShape s;
    if (!plan_of(joined, a, type, ctx, &s)) return kBadArgument;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return joined ? run<T, true>(a, s, ctx, st) : run<T, false>(a, s, ctx, st);
    });
}

}  // namespace ldn
