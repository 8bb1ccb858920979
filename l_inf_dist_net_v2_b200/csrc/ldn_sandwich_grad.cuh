// The residual stream between two norms, backward, with rows in registers (ldn_sandwich_rows.cuh).
#pragma once
#include "ldn_sandwich_rows.cuh"

namespace ldn {
namespace {

template <int N>
__device__ __forceinline__ float at_of(const float2 (&v)[N], int e) {
    return e % 2 ? v[e / 2].y : v[e / 2].x;
}

// OF_Y: a gradient of y comes; without it neither h nor its statistics are read (what they are does not matter then, infinities neither): one round
// of sums and two streams fewer, 16384 x 5120 bf16 with a gate of its shape 175 us where both gradients take 287.
template <class T, Gate G, int ITEMS, Share W, bool SHIFT, bool OF_Y>
__global__ void __launch_bounds__(W == Share::Group ? kGroupThreads : most_threads(ITEMS * kPiece<T>), 1)
sandwich_grad_registers_kernel(const __grid_constant__ SandwichGradArgs a, int lanes, int depth, int ranks) {
    stream_order_begin();
    constexpr bool GROUP = W == Share::Group;
    constexpr int V = kPiece<T>, S = kBackwardStreams<G, OF_Y>, R = 1;
    constexpr int kOfH = 1, kOfDy = 2, kOfDh = OF_Y ? 3 : 1, kOfGate = OF_Y ? 4 : 2;  // streams' numbers (x has 0)
    constexpr int K = G == Gate::Row ? 4 : 2;  // sums of a row in the second round (a power of two)
    __shared__ alignas(16) float slots[2 * SumOf<W>::kSlots];
    extern __shared__ uint4 ring[];  // [depth][row][stream][item][thread], then blocks: [3][item][V / 4][thread]; at the end, groups: [warp][4][C] floats
    const int rank = W == Share::Cluster ? static_cast<int>(cluster_rank()) : 0;
    SumOf<W> reduce{lanes, slots, 0, ranks, rank};
    reduce.begin();
    const int lane = GROUP ? threadIdx.x & (lanes - 1) : rank * blockDim.x + threadIdx.x;
    const int per_block = GROUP ? kGroupThreads / lanes : 1;
    const unsigned block = W == Share::Cluster ? blockIdx.x / ranks : blockIdx.x, blocks = W == Share::Cluster ? gridDim.x / ranks : gridDim.x;
    const long long step = static_cast<long long>(blocks) * per_block;
    const long long mine = static_cast<long long>(block) * per_block + (GROUP ? threadIdx.x / lanes : 0);
    const float inv_C = 1.0f / a.C;
    const int shift = SHIFT ? shift_of(static_cast<const T*>(a.x) + (mine < a.rows ? mine : 0) * a.pitch) : 0;
    auto column = [&](int i) { return (lane + i * lanes) * V - shift; };
    // a group's columns' parameters stay in registers, a block's in shared memory, where each thread puts and finds its own (as registers, the
    // kernel spilled: 16384 x 5120 bf16 415 us)
    float2 kept[GROUP ? 3 : 1][GROUP ? ITEMS : 1][V / 2];
    uint4* params = ring + static_cast<size_t>(depth) * R * S * ITEMS * blockDim.x + threadIdx.x;
    auto set_param_piece = [&](int k, int i, const float2 (&v)[V / 2]) {
#pragma unroll
        for (int e = 0; e < V / 2; e += 2) {
            if constexpr (GROUP) {
                kept[k][i][e] = v[e];
                kept[k][i][e + 1] = v[e + 1];
            } else {
                params[((k * ITEMS + i) * (V / 4) + e / 2) * blockDim.x] =
                    make_uint4(__float_as_uint(v[e].x), __float_as_uint(v[e].y), __float_as_uint(v[e + 1].x), __float_as_uint(v[e + 1].y));
            }
        }
    };
    auto param_piece = [&](int k, int i, float2 (&v)[V / 2]) {
#pragma unroll
        for (int e = 0; e < V / 2; e += 2) {
            if constexpr (GROUP) {
                v[e] = kept[k][i][e];
                v[e + 1] = kept[k][i][e + 1];
            } else {
                const uint4 raw = params[((k * ITEMS + i) * (V / 4) + e / 2) * blockDim.x];
                v[e] = make_float2(__uint_as_float(raw.x), __uint_as_float(raw.y));
                v[e + 1] = make_float2(__uint_as_float(raw.z), __uint_as_float(raw.w));
            }
        }
    };
    float2 sums[4][ITEMS][V / 2];  // dy z2, dy, d gate z1, d gate
    uint4 mask[ITEMS];
    int bytes[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < V / 2; ++e) sums[k][i][e] = both(0.0f);
        mask[i] = mask_of<T, SHIFT>(column(i), a.C);
        bytes[i] = piece_bytes<T>(column(i), a.C);
        float2 w[V / 2], b[V / 2];
        load_scaled<T, SHIFT>(a.p, column(i), a.C, w, b);
        set_param_piece(0, i, w);
        set_param_piece(1, i, b);
        load_params<T, SHIFT>(a.p.weight, a.p.wide, column(i), a.C, 1.0f, w);
        set_param_piece(2, i, w);
    }
    const int c0 = column(0), apart = lanes * V;
    int to_fetch = mine < a.rows ? static_cast<int>((a.rows - mine + step - 1) / step) : 0, to_make = to_fetch;
    Walk<const T> from_x(a.x, a.pitch, mine, step, c0), from_h(a.h, a.C, mine, step, c0), from_dy(a.grad_y, a.C, mine, step, c0),
        from_dh(a.grad_h, a.C, mine, step, c0), from_gate(a.gate, G == Gate::All ? a.pitch_gate : 0, mine, step, c0);
    Walk<T> to_x(a.grad_x, a.C, mine, step, c0), to_onto(a.grad_residual, a.C, mine, step, c0), to_gate(a.grad_gate, a.C, mine, step, c0);
    long long row0 = mine;
    uint4* own = ring + threadIdx.x;
    auto slot_of = [&](int stage, int j, int stream, int i) { return own + (((stage * R + j) * S + stream) * ITEMS + i) * blockDim.x; };
    auto fetch = [&](int stage) {
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (j < to_fetch) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    copy_piece<T, SHIFT>(slot_of(stage, j, 0, i), from_x.of(j, i * apart), column(i), bytes[i], a.x);
                    if constexpr (OF_Y) {
                        copy_piece<T, SHIFT>(slot_of(stage, j, kOfH, i), from_h.of(j, i * apart), column(i), bytes[i], a.h);
                        // (asked for although it comes: the compiler's order without is slower, 9999 x 1001 f16 87 us instead of 81)
                        if (a.grad_y) copy_piece<T, SHIFT>(slot_of(stage, j, kOfDy, i), from_dy.of(j, i * apart), column(i), bytes[i], a.grad_y);
                    }
                    if (a.grad_h) copy_piece<T, SHIFT>(slot_of(stage, j, kOfDh, i), from_dh.of(j, i * apart), column(i), bytes[i], a.grad_h);
                    if constexpr (G == Gate::All)
                        copy_piece<T, SHIFT>(slot_of(stage, j, kOfGate, i), from_gate.of(j, i * apart), column(i), bytes[i], a.gate);
                }
            }
        copies_commit();
        to_fetch -= R;
        from_x.on(R);
        if constexpr (OF_Y) {
            from_h.on(R);
            from_dy.on(R);
        }
        from_dh.on(R);
        if constexpr (G == Gate::All) from_gate.on(R);
    };
    // (zeros for pieces behind the row's end, and for a gradient that does not come)
    for (int d = 0; d < depth * R * S; ++d)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (!bytes[i] || (OF_Y && !a.grad_y && d % S == kOfDy) || (!a.grad_h && d % S == kOfDh)) own[(d * ITEMS + i) * blockDim.x] = make_uint4(0u, 0u, 0u, 0u);
    for (int d = 0; d < depth; ++d) fetch(d);
    constexpr int kStats = OF_Y ? 4 : 2, kNumbers = G == Gate::Row ? kStats + 1 : kStats;
    __shared__ float numbers[kNumbers][kNumberRows];
    int stage = 0;
    const long long block_first = static_cast<long long>(block) * per_block;
    const int turns = block_first < a.rows ? static_cast<int>((a.rows - block_first + R * step - 1) / (R * step)) : 0;
    auto row_of = [&](int turn, int i) { return block_first + (static_cast<long long>(turn) * R + i / per_block) * step + i % per_block; };
    for (int turn = 0; turn < turns; ++turn) {
        auto live = [&](int j) { return j < to_make; };
        float mean1[R], rstd1[R], mean2[R], rstd2[R], gate[R], s[2 * R], t[K * R];
        RowNumbers<kNumbers, R * kNumberRows> of_rows(numbers, R * per_block);
        of_rows.at_turn(turn, a.rows, [&](int i) { return row_of(turn, i); }, [&](int k, long long row) {
            return k < kStats ? a.stats[k * a.rows + row] : to_float(static_cast<const T*>(a.gate)[row]);
        });
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int index = j * per_block + (GROUP ? threadIdx.x / lanes : 0);
            mean1[j] = of_rows.of(0, turn, index);
            rstd1[j] = of_rows.of(1, turn, index);
            mean2[j] = OF_Y ? of_rows.of(2, turn, index) : 0.0f;
            rstd2[j] = OF_Y ? of_rows.of(3, turn, index) : 0.0f;
            gate[j] = G == Gate::Row ? of_rows.of(kNumbers - 1, turn, index) : 1.0f;
        }
        copies_wait(depth);
        // (outside the row all is 0)
        auto piece_of = [&](int j, int stream, int i, float2 (&v)[V / 2]) {
            const uint4 raw = live(j) ? *slot_of(stage, j, stream, i) : make_uint4(0u, 0u, 0u, 0u);
            unpack<T>(SHIFT ? masked(raw, mask[i]) : raw, v);
        };
        if constexpr (OF_Y) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    float2 h[V / 2], dy[V / 2], w2[V / 2];
                    piece_of(j, kOfH, i, h);
                    piece_of(j, kOfDy, i, dy);
                    param_piece(2, i, w2);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        // (rstd behind the sum: outside the row the gradient is 0 and h - mean a number, but (0 - mean) rstd may be infinite)
                        const float2 u = __fmul2_rn(dy[e], __fadd2_rn(h[e], both(-mean2[j])));
                        sums[0][i][e] = __ffma2_rn(u, both(rstd2[j]), sums[0][i][e]);
                        sums[1][i][e] = __fadd2_rn(sums[1][i][e], dy[e]);
                        s0 = __ffma2_rn(dy[e], w2[e], s0);
                        s1 = __ffma2_rn(u, w2[e], s1);
                    }
                }
                s[2 * j] = s0.x + s0.y;
                s[2 * j + 1] = s1.x + s1.y;
            }
            reduce(s, [&](float all) { return all * inv_C; });
        }
        float2 by[R][ITEMS][V / 2];  // what goes into the first norm's gradient
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float2 t0 = both(0.0f), t1 = both(0.0f), tg = both(0.0f);
            const float m1 = OF_Y ? s[2 * j] : 0.0f, m2 = OF_Y ? s[2 * j + 1] * rstd2[j] * rstd2[j] : 0.0f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = column(i);
                float2 d[V / 2], h[V / 2], x[V / 2], n[V / 2], w[V / 2];
                if constexpr (OF_Y) {
                    piece_of(j, kOfH, i, h);
                    piece_of(j, kOfDy, i, d);
                    param_piece(2, i, w);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e)
                        d[e] = __ffma2_rn(__fadd2_rn(h[e], both(-mean2[j])), both(-m2), __ffma2_rn(d[e], w[e], both(-m1)));
                }
                piece_of(j, kOfDh, i, h);
                piece_of(j, 0, i, x);
                param_piece(0, i, w);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    d[e] = OF_Y ? __ffma2_rn(d[e], both(rstd2[j]), h[e]) : h[e];
                    x[e] = __fadd2_rn(x[e], both(-mean1[j]));  // (rstd behind the sums, as above)
                }
                if (live(j) && a.grad_residual) store_piece<T, SHIFT>(to_onto.of(j, i * apart), c, a.C, pack<T>(d));
                if constexpr (G != Gate::None) {
                    param_piece(1, i, n);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) n[e] = __fmul2_rn(d[e], __ffma2_rn(__fmul2_rn(x[e], both(rstd1[j])), w[e], n[e]));
                }
                if constexpr (G == Gate::All) {
                    if (live(j) && a.grad_gate) store_piece<T, SHIFT>(to_gate.of(j, i * apart), c, a.C, pack<T>(n));
                    float2 g[V / 2];
                    piece_of(j, kOfGate, i, g);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) d[e] = __fmul2_rn(d[e], g[e]);
                } else if constexpr (G == Gate::Row) {
                    only_row<SHIFT>(c, a.C, n);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        tg = __fadd2_rn(tg, n[e]);
                        d[e] = __fmul2_rn(d[e], both(gate[j]));
                    }
                }
                only_row<SHIFT>(c, a.C, d);
                if (!live(j))
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) d[e] = both(0.0f);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 u = __fmul2_rn(d[e], x[e]);
                    sums[2][i][e] = __ffma2_rn(u, both(rstd1[j]), sums[2][i][e]);
                    sums[3][i][e] = __fadd2_rn(sums[3][i][e], d[e]);
                    by[j][i][e] = __fmul2_rn(d[e], w[e]);
                    t0 = __fadd2_rn(t0, by[j][i][e]);
                    t1 = __ffma2_rn(u, w[e], t1);
                }
            }
            t[K * j] = t0.x + t0.y;
            t[K * j + 1] = t1.x + t1.y;
            if constexpr (G == Gate::Row) {
                t[K * j + 2] = tg.x + tg.y;
                t[K * j + 3] = 0.0f;
            }
        }
        reduce(t, [&](float all) { return all; });
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (!live(j)) continue;
            if constexpr (G == Gate::Row)
                if (lane == 0 && a.grad_gate) static_cast<T*>(a.grad_gate)[row0 + j * step] = from_float<T>(t[K * j + 2]);
            if (!a.grad_x) continue;
            const float m1 = t[K * j] * inv_C, m2 = t[K * j + 1] * inv_C * rstd1[j] * rstd1[j];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                float2 x[V / 2];
                piece_of(j, 0, i, x);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 p = __fadd2_rn(by[j][i][e], both(-m1));
                    x[e] = __fmul2_rn(__ffma2_rn(__fadd2_rn(x[e], both(-mean1[j])), both(-m2), p), both(rstd1[j]));
                }
                store_piece<T, SHIFT>(to_x.of(j, i * apart), column(i), a.C, pack<T>(x));
            }
        }
        fetch(stage);
        stage = stage + 1 == depth ? 0 : stage + 1;
        to_make -= R;
        row0 += R * step;
        to_x.on(R);
        to_onto.on(R);
        to_gate.on(R);
    }
    if constexpr (W == Share::Cluster) cluster_barrier();  // (no block ends while another may still write to it)
    if (!a.parts) return;
    float* part = a.parts + static_cast<long long>(block) * 4 * a.C;
    if constexpr (!GROUP) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = column(i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (!SHIFT) {
                    if (c >= a.C) continue;
#pragma unroll
                    for (int e = 0; e < V / 2; e += 2)
                        *reinterpret_cast<float4*>(part + k * a.C + c + 2 * e) =
                            make_float4(sums[k][i][e].x, sums[k][i][e].y, sums[k][i][e + 1].x, sums[k][i][e + 1].y);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (static_cast<unsigned>(c + e) < static_cast<unsigned>(a.C)) part[k * a.C + c + e] = at_of(sums[k][i], e);
                }
            }
        }
    } else {
        // a warp's groups add to its columns in turn, then the warps' are added up
        float* columns = reinterpret_cast<float*>(ring);
        copies_wait(1);
        __syncthreads();  // (all have read their rows)
        float* own = columns + (threadIdx.x >> 5) * 4 * a.C;
        const int turn = (threadIdx.x & 31) / lanes;
        for (int q = 0; q < 32 / lanes; ++q) {
            if (turn == q)
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int c = column(i) + e;
                        if (static_cast<unsigned>(c) < static_cast<unsigned>(a.C))
#pragma unroll
                            for (int k = 0; k < 4; ++k) own[k * a.C + c] = at_of(sums[k][i], e) + (q ? own[k * a.C + c] : 0.0f);
                    }
            __syncwarp();
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 4 * a.C; c += kGroupThreads) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kGroupThreads / 32; ++w) s += columns[w * 4 * a.C + c];
            part[c] = s;
        }
    }
}

bool plan_backward(Gate gate, const SandwichGradArgs& a, int size, RowPlan* p, Share* who, int* ranks) {
    const bool aligned = on16(a.x) && on16(a.h) && on16(a.grad_y) && on16(a.grad_h) && on16(a.grad_x) && on16(a.grad_residual) &&
                         (gate != Gate::All || (on16(a.gate) && on16(a.grad_gate)));
    const bool match = rows_match(size, a.C, a.pitch, aligned) && (gate != Gate::All || rows_match(size, a.C, a.pitch_gate, aligned));
    const bool shift = rows_shift(size, a.C) || !on16(a.p.scale) || !on16(a.p.post_weight) || !on16(a.p.post_bias) || !on16(a.p.weight);
    return match && plan_row(a.C, size, shift, false, p, who, ranks);
}
// The backward kernel for these rows, with its shape: f(kernel, shape); kBadArgument where there is none
template <class T, bool OF_Y, class F>
int with_backward(Gate gate, const SandwichGradArgs& a, const DeviceCtx* ctx, F f) {
    RowPlan p;
    Share who;
    int ranks;
    if (!plan_backward(gate, a, sizeof(T), &p, &who, &ranks)) return kBadArgument;
    return with_gate(gate, [&](auto g) {
        return with_items<T, false>(p, who, [&](auto items, auto share, auto shift) {
            constexpr Gate G = decltype(g)::value;
            constexpr int kItems = decltype(items)::value;
            constexpr Share W = decltype(share)::value;
            constexpr auto kernel = sandwich_grad_registers_kernel<T, G, kItems, W, decltype(shift)::value, OF_Y>;
            const long long params = W == Share::Group ? 0 : 3LL * kItems * (kPiece<T> / 4) * p.threads * 16;
            long long resident;
            int depth;
            RowShape s;
            if (!resident_rows<kernel, W>(p, 1, kBackwardStreams<G, OF_Y>, params, ranks, ctx, &resident, &depth) ||
                !shape_of(p, a.rows, 1, kBackwardStreams<G, OF_Y>, params, ranks, resident, depth, &s))
                return static_cast<int>(kBadArgument);
            if constexpr (W == Share::Group) {
                const size_t columns = static_cast<size_t>(kGroupThreads / 32) * 4 * a.C * sizeof(float);
                if (s.smem < columns) s.smem = columns;
            }
            return f(kernel, s);
        });
    });
}

}  // namespace

template <class T, bool OF_Y>
int sandwich_grad_rows(Gate gate, const SandwichGradArgs& a, const DeviceCtx* ctx, int* blocks, const cudaStream_t* st) {
    return with_backward<T, OF_Y>(gate, a, ctx, [&](auto kernel, const RowShape& s) {
        if (blocks) *blocks = s.blocks;
        if (!st) return static_cast<int>(kOk);
        return launch_after_in_clusters(kernel, s.ranks, s.blocks * s.ranks, s.p.threads, s.smem, *st, a, s.p.lanes, s.depth, s.ranks);
    });
}

}  // namespace ldn
