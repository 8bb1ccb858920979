// The residual stream between two norms, forward, with rows in registers (ldn_sandwich_rows.cuh).
#pragma once
#include "ldn_sandwich_rows.cuh"

namespace ldn {
namespace {

template <class T, Gate G, int ITEMS, Share W, bool SHIFT>
__global__ void __launch_bounds__(W == Share::Group ? kGroupThreads : most_threads(ITEMS * kPiece<T>), 1)
sandwich_registers_kernel(const __grid_constant__ SandwichArgs a, int lanes, int depth, int ranks) {
    stream_order_begin();
    constexpr bool GROUP = W == Share::Group, kKeep = ITEMS * kPiece<T> <= 16;  // (the columns' parameters stay in registers)
    constexpr int V = kPiece<T>, S = kForwardStreams<G>, R = rows_forward(ITEMS * V);
    __shared__ alignas(16) float slots[2 * SumOf<W>::kSlots];
    extern __shared__ uint4 ring[];  // [depth][row][stream][item][thread]
    const int rank = W == Share::Cluster ? static_cast<int>(cluster_rank()) : 0;
    SumOf<W> reduce{lanes, slots, 0, ranks, rank};
    reduce.begin();
    const int lane = GROUP ? threadIdx.x & (lanes - 1) : rank * blockDim.x + threadIdx.x;
    const int per_block = GROUP ? kGroupThreads / lanes : 1;
    const unsigned block = W == Share::Cluster ? blockIdx.x / ranks : blockIdx.x, blocks = W == Share::Cluster ? gridDim.x / ranks : gridDim.x;
    const long long step = static_cast<long long>(blocks) * per_block;
    const long long mine = static_cast<long long>(block) * per_block + (GROUP ? threadIdx.x / lanes : 0);
    const float inv_C = 1.0f / a.C;
    // (the same for all rows of this thread)
    const int shift = SHIFT ? shift_of(static_cast<const T*>(a.x) + (mine < a.rows ? mine : 0) * a.pitch) : 0;
    auto column = [&](int i) { return (lane + i * lanes) * V - shift; };
    float2 w1[ITEMS][V / 2], b1[ITEMS][V / 2], w2[ITEMS][V / 2], b2[ITEMS][V / 2];
    uint4 mask[ITEMS];
    int bytes[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        mask[i] = mask_of<T, SHIFT>(column(i), a.C);
        bytes[i] = piece_bytes<T>(column(i), a.C);
        if constexpr (kKeep) {
            load_scaled<T, SHIFT>(a.p, column(i), a.C, w1[i], b1[i]);
            load_params<T, SHIFT>(a.p.weight, a.p.wide, column(i), a.C, 1.0f, w2[i]);
            load_params<T, SHIFT>(a.p.bias, a.p.wide, column(i), a.C, 0.0f, b2[i]);
        }
    }
    const int c0 = column(0), apart = lanes * V;
    int to_fetch = mine < a.rows ? static_cast<int>((a.rows - mine + step - 1) / step) : 0, to_make = to_fetch;
    Walk<const T> from_x(a.x, a.pitch, mine, step, c0), from_onto(a.residual, a.pitch_residual, mine, step, c0),
        from_gate(a.gate, G == Gate::All ? a.pitch_gate : 0, mine, step, c0);
    Walk<T> to_h(a.h, a.C, mine, step, c0), to_y(a.y, a.C, mine, step, c0);
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
                    copy_piece<T, SHIFT>(slot_of(stage, j, 1, i), from_onto.of(j, i * apart), column(i), bytes[i], a.residual);
                    if constexpr (G == Gate::All)
                        copy_piece<T, SHIFT>(slot_of(stage, j, 2, i), from_gate.of(j, i * apart), column(i), bytes[i], a.gate);
                }
            }
        copies_commit();
        to_fetch -= R;
        from_x.on(R);
        from_onto.on(R);
        if constexpr (G == Gate::All) from_gate.on(R);
    };
    for (int d = 0; d < depth * R * S; ++d)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (!bytes[i]) own[(d * ITEMS + i) * blockDim.x] = make_uint4(0u, 0u, 0u, 0u);
    for (int d = 0; d < depth; ++d) fetch(d);
    __shared__ float numbers[1][G == Gate::Row ? R * kNumberRows : 1];
    int stage = 0;
    // (a warp's groups take part in its shuffles whether they have a row or not: as many turns as the block's first has)
    const long long block_first = static_cast<long long>(block) * per_block;
    const int turns = block_first < a.rows ? static_cast<int>((a.rows - block_first + R * step - 1) / (R * step)) : 0;
    auto row_of = [&](int turn, int i) { return block_first + (static_cast<long long>(turn) * R + i / per_block) * step + i % per_block; };
    for (int turn = 0; turn < turns; ++turn) {
        auto live = [&](int j) { return j < to_make; };
        float gate[R];
        if constexpr (G == Gate::Row) {
            RowNumbers<1, R * kNumberRows> gates(numbers, R * per_block);
            gates.at_turn(turn, a.rows, [&](int i) { return row_of(turn, i); },
                          [&](int, long long row) { return to_float(static_cast<const T*>(a.gate)[row]); });
#pragma unroll
            for (int j = 0; j < R; ++j) gate[j] = gates.of(0, turn, j * per_block + (GROUP ? threadIdx.x / lanes : 0));
        }
        copies_wait(depth);
        float2 v[R][ITEMS][V / 2];
        float s[R], mean[R];
        auto piece_of = [&](int j, int stream, int i) { return live(j) ? *slot_of(stage, j, stream, i) : make_uint4(0u, 0u, 0u, 0u); };
#pragma unroll
        for (int j = 0; j < R; ++j) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const uint4 raw = piece_of(j, 0, i);
                unpack<T>(SHIFT ? masked(raw, mask[i]) : raw, v[j][i]);
            }
        }
        // mean and deviation of what the registers hold: v becomes v - mean, s 1 / deviation
        auto statistics = [&](float* to) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                float2 sum = both(0.0f);
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) sum = __fadd2_rn(sum, v[j][i][e]);
                s[j] = sum.x + sum.y;
            }
            reduce(s, [&](float all) { return all * inv_C; });
#pragma unroll
            for (int j = 0; j < R; ++j) {
                mean[j] = s[j];
                float2 sum = both(0.0f);
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) v[j][i][e] = __fadd2_rn(v[j][i][e], both(-mean[j]));
                    only_row<SHIFT>(column(i), a.C, v[j][i]);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) sum = __ffma2_rn(v[j][i][e], v[j][i][e], sum);
                }
                s[j] = sum.x + sum.y;
            }
            reduce(s, [&](float all) { return 1.0f / sqrtf(all * inv_C + a.eps); });
            if (lane == 0 && a.stats)
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (live(j)) {
                        to[row0 + j * step] = mean[j];
                        to[a.rows + row0 + j * step] = s[j];
                    }
        };
        statistics(a.stats);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = column(i);
            if constexpr (!kKeep) load_scaled<T, SHIFT>(a.p, c, a.C, w1[i], b1[i]);
#pragma unroll
            for (int j = 0; j < R; ++j) {
                float2 onto[V / 2], g[V / 2];
                unpack<T>(piece_of(j, 1, i), onto);
                if constexpr (G == Gate::All) unpack<T>(piece_of(j, 2, i), g);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 n = __ffma2_rn(__fmul2_rn(v[j][i][e], both(s[j])), w1[i][e], b1[i][e]);
                    v[j][i][e] = G == Gate::None ? __fadd2_rn(onto[e], n) : __ffma2_rn(G == Gate::All ? g[e] : both(gate[j]), n, onto[e]);
                }
                uint4 raw = pack<T>(v[j][i]);
                if (live(j)) store_piece<T, SHIFT>(to_h.of(j, i * apart), c, a.C, raw);
                if (!SHIFT && c >= a.C) raw = make_uint4(0u, 0u, 0u, 0u);
                unpack<T>(SHIFT ? masked(raw, mask[i]) : raw, v[j][i]);
            }
        }
        fetch(stage);
        stage = stage + 1 == depth ? 0 : stage + 1;
        statistics(a.stats + 2 * a.rows);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = column(i);
            if constexpr (!kKeep) {
                load_params<T, SHIFT>(a.p.weight, a.p.wide, c, a.C, 1.0f, w2[i]);
                load_params<T, SHIFT>(a.p.bias, a.p.wide, c, a.C, 0.0f, b2[i]);
            }
#pragma unroll
            for (int j = 0; j < R; ++j) {
#pragma unroll
                for (int e = 0; e < V / 2; ++e) v[j][i][e] = __ffma2_rn(__fmul2_rn(v[j][i][e], both(s[j])), w2[i][e], b2[i][e]);
                if (live(j)) store_piece<T, SHIFT>(to_y.of(j, i * apart), c, a.C, pack<T>(v[j][i]));
            }
        }
        to_make -= R;
        row0 += R * step;
        to_h.on(R);
        to_y.on(R);
    }
    if constexpr (W == Share::Cluster) cluster_barrier();  // (no block ends while another may still write to it)
}

bool plan_forward(Gate gate, const SandwichArgs& a, int size, RowPlan* p, Share* who, int* ranks) {
    const bool aligned = on16(a.x) && on16(a.residual) && on16(a.h) && on16(a.y) && (gate != Gate::All || on16(a.gate));
    const bool match = rows_match(size, a.C, a.pitch, aligned) && rows_match(size, a.C, a.pitch_residual, aligned) &&
                       (gate != Gate::All || rows_match(size, a.C, a.pitch_gate, aligned));
    const bool shift = rows_shift(size, a.C) || !on16(a.p.scale) || !on16(a.p.post_weight) || !on16(a.p.post_bias) || !on16(a.p.weight) ||
                       !on16(a.p.bias);
    return match && plan_row(a.C, size, shift, true, p, who, ranks);
}
}  // namespace

template <class T>
bool sandwich_rows(Gate gate, const SandwichArgs& a, const DeviceCtx* ctx, cudaStream_t st, int* status) {
    RowPlan p;
    Share who;
    int ranks;
    if (!plan_forward(gate, a, sizeof(T), &p, &who, &ranks)) return false;
    bool fits = false;
    *status = with_gate(gate, [&](auto g) {
        return with_items<T, true>(p, who, [&](auto items, auto share, auto shift) {
            constexpr Gate G = decltype(g)::value;
            constexpr int kItems = decltype(items)::value;
            constexpr Share W = decltype(share)::value;
            constexpr auto kernel = sandwich_registers_kernel<T, G, kItems, W, decltype(shift)::value>;
            constexpr int R = rows_forward(kItems * kPiece<T>);
            long long resident;
            int depth;
            RowShape s;
            fits = resident_rows<kernel, W>(p, R, kForwardStreams<G>, 0, ranks, ctx, &resident, &depth) &&
                   shape_of(p, a.rows, R, kForwardStreams<G>, 0, ranks, resident, depth, &s);
            return fits ? launch_after_in_clusters(kernel, ranks, s.blocks * ranks, p.threads, s.smem, st, a, p.lanes, s.depth, ranks)
                        : static_cast<int>(kOk);
        });
    });
    return fits;
}

}  // namespace ldn
