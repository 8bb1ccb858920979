// The residual stream between two norms with rows in registers: forward one read of x, the residual and the gate and four sums over a row,
// backward one read of the five tensors that it takes and two rounds of sums, with the column sums carried in the threads that have those
// columns, from row to row.
//
// Bound by memory.  As in the layer norm's kernels, rows are under way into shared memory while others are summed, a block takes every
// gridDim-th row, so that its threads' columns and parameters stay (rows that start anywhere in 16 bytes: the grid is a multiple of
// eight, and rows that far apart start alike), and rows that are taken together share the barriers of their sums.  The scale and the first
// norm's parameters are two numbers per column, scale weight and scale bias.
#include "ldn_sandwich.cuh"
#include "ldn_rows.cuh"

namespace ldn {
namespace {

template <Gate G>
constexpr int kForwardStreams = G == Gate::All ? 3 : 2;
template <Gate G>
constexpr int kBackwardStreams = G == Gate::All ? 5 : 4;
// Rows that a block, or each of its groups, takes at a time forward; backward one (524288 x 96 bf16 with a gate per row, 1 / 2 / 4 rows of a
// group: 172 / 145 / 131 us, backward 236 / 306; 1000000 x 17, cut rows: 107 / 111 / 141; 200000 x 40 f32: 45 / 43 / 49)
__host__ __device__ constexpr int rows_forward(int elements, int size, bool group, bool shift) {
    return group ? (elements <= 8 && size == 2 && !shift ? 4 : 2) : elements > 16 ? 1 : 2;
}

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
template <bool GROUP>
struct SumOf {
    int lanes;
    float* slots;  // [2][kSlots], zeros at first
    int turn;
    static constexpr int kSlots = 20 * 8;  // (warps of a block) x K, a multiple of four numbers
    __device__ __forceinline__ void begin() {
        if constexpr (!GROUP)
            for (int i = threadIdx.x; i < 2 * kSlots; i += blockDim.x) slots[i] = 0.0f;
        __syncthreads();
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
            if (lane % kShare == 0) s[(threadIdx.x >> 5) * K + lane / kShare] = v[0];
            __syncthreads();
            const int pieces = (static_cast<int>(blockDim.x >> 5) * K + 3) / 4;
            const float4* from = reinterpret_cast<const float4*>(s);
            if constexpr (K == 8) {
                float4 a = from[0], b = from[1];
                for (int i = 2; i < pieces; i += 2) {
                    const float4 c = from[i], d = from[i + 1];
                    a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
                    b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
                }
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            } else {
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
            }
#pragma unroll
            for (int i = 0; i < K; ++i) v[i] = end(v[i]);
        }
    }
};

template <class T, Gate G, int ITEMS, bool GROUP, bool SHIFT>
__global__ void __launch_bounds__(GROUP ? kGroupThreads : threads_of(ITEMS * kPiece<T>), 1)
sandwich_registers_kernel(const __grid_constant__ SandwichArgs a, int lanes, int depth) {
    stream_order_begin();
    constexpr int V = kPiece<T>, S = kForwardStreams<G>, R = rows_forward(ITEMS * V, sizeof(T), GROUP, SHIFT);
    constexpr bool kKeep = ITEMS * V <= 16;
    __shared__ alignas(16) float slots[2 * SumOf<GROUP>::kSlots];
    extern __shared__ uint4 ring[];  // [depth][row][stream][item][thread]
    SumOf<GROUP> reduce{lanes, slots, 0};
    reduce.begin();
    const int lane = GROUP ? threadIdx.x & (lanes - 1) : threadIdx.x;
    const int per_block = GROUP ? kGroupThreads / lanes : 1;
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    const long long mine = static_cast<long long>(blockIdx.x) * per_block + (GROUP ? threadIdx.x / lanes : 0);
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
    const long long block_first = static_cast<long long>(blockIdx.x) * per_block;
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
}

template <int N>
__device__ __forceinline__ float at_of(const float2 (&v)[N], int e) {
    return e % 2 ? v[e / 2].y : v[e / 2].x;
}

template <class T, Gate G, int ITEMS, bool GROUP, bool SHIFT>
__global__ void __launch_bounds__(GROUP ? kGroupThreads : threads_of(ITEMS * kPiece<T>), 1)
sandwich_grad_registers_kernel(const __grid_constant__ SandwichGradArgs a, int lanes, int depth) {
    stream_order_begin();
    constexpr int V = kPiece<T>, S = kBackwardStreams<G>, R = 1;
    constexpr bool kSums = ITEMS * V <= 16;  // (rows of 32 elements per thread leave their column sums to a kernel of its own)
    constexpr int K = G == Gate::Row ? 4 : 2;  // sums of a row in the second round (a power of two)
    __shared__ alignas(16) float slots[2 * SumOf<GROUP>::kSlots];
    extern __shared__ uint4 ring[];  // [depth][row][stream][item][thread], then blocks: [3][item][V / 4][thread]; at the end, groups: [warp][4][C] floats
    SumOf<GROUP> reduce{lanes, slots, 0};
    reduce.begin();
    const int lane = GROUP ? threadIdx.x & (lanes - 1) : threadIdx.x;
    const int per_block = GROUP ? kGroupThreads / lanes : 1;
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    const long long mine = static_cast<long long>(blockIdx.x) * per_block + (GROUP ? threadIdx.x / lanes : 0);
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
    auto param_piece = [&](int k, int i, int first, float2 (&v)[V / 2]) {
        if constexpr (!kSums) {
            float2 other[V / 2];
            if (k == 2) load_params<T, SHIFT>(a.p.weight, a.p.wide, first, a.C, 1.0f, v);
            else if (k == 1) load_scaled<T, SHIFT>(a.p, first, a.C, other, v);
            else load_scaled<T, SHIFT>(a.p, first, a.C, v, other);
        } else {
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
        }
    };
    float2 sums[4][kSums ? ITEMS : 1][V / 2];  // dy z2, dy, d gate z1, d gate
    uint4 mask[ITEMS];
    int bytes[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if constexpr (kSums)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < V / 2; ++e) sums[k][i][e] = both(0.0f);
        mask[i] = mask_of<T, SHIFT>(column(i), a.C);
        bytes[i] = piece_bytes<T>(column(i), a.C);
        if constexpr (kSums) {
            float2 w[V / 2], b[V / 2];
            load_scaled<T, SHIFT>(a.p, column(i), a.C, w, b);
            set_param_piece(0, i, w);
            set_param_piece(1, i, b);
            load_params<T, SHIFT>(a.p.weight, a.p.wide, column(i), a.C, 1.0f, w);
            set_param_piece(2, i, w);
        }
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
                    copy_piece<T, SHIFT>(slot_of(stage, j, 1, i), from_h.of(j, i * apart), column(i), bytes[i], a.h);
                    if (a.grad_y) copy_piece<T, SHIFT>(slot_of(stage, j, 2, i), from_dy.of(j, i * apart), column(i), bytes[i], a.grad_y);
                    if (a.grad_h) copy_piece<T, SHIFT>(slot_of(stage, j, 3, i), from_dh.of(j, i * apart), column(i), bytes[i], a.grad_h);
                    if constexpr (G == Gate::All)
                        copy_piece<T, SHIFT>(slot_of(stage, j, 4, i), from_gate.of(j, i * apart), column(i), bytes[i], a.gate);
                }
            }
        copies_commit();
        to_fetch -= R;
        from_x.on(R);
        from_h.on(R);
        from_dy.on(R);
        from_dh.on(R);
        if constexpr (G == Gate::All) from_gate.on(R);
    };
    // (zeros for pieces behind the row's end, and for a gradient that does not come)
    for (int d = 0; d < depth * R * S; ++d)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (!bytes[i] || (!a.grad_y && d % S == 2) || (!a.grad_h && d % S == 3)) own[(d * ITEMS + i) * blockDim.x] = make_uint4(0u, 0u, 0u, 0u);
    for (int d = 0; d < depth; ++d) fetch(d);
    constexpr int kNumbers = G == Gate::Row ? 5 : 4;
    __shared__ float numbers[kNumbers][kNumberRows];
    int stage = 0;
    const long long block_first = static_cast<long long>(blockIdx.x) * per_block;
    const int turns = block_first < a.rows ? static_cast<int>((a.rows - block_first + R * step - 1) / (R * step)) : 0;
    auto row_of = [&](int turn, int i) { return block_first + (static_cast<long long>(turn) * R + i / per_block) * step + i % per_block; };
    for (int turn = 0; turn < turns; ++turn) {
        auto live = [&](int j) { return j < to_make; };
        float mean1[R], rstd1[R], mean2[R], rstd2[R], gate[R], s[2 * R], t[K * R];
        RowNumbers<kNumbers, R * kNumberRows> of_rows(numbers, R * per_block);
        of_rows.at_turn(turn, a.rows, [&](int i) { return row_of(turn, i); }, [&](int k, long long row) {
            return k < 4 ? a.stats[k * a.rows + row] : to_float(static_cast<const T*>(a.gate)[row]);
        });
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int index = j * per_block + (GROUP ? threadIdx.x / lanes : 0);
            mean1[j] = of_rows.of(0, turn, index);
            rstd1[j] = of_rows.of(1, turn, index);
            mean2[j] = of_rows.of(2, turn, index);
            rstd2[j] = of_rows.of(3, turn, index);
            gate[j] = G == Gate::Row ? of_rows.of(kNumbers - 1, turn, index) : 1.0f;
        }
        copies_wait(depth);
        // (outside the row all is 0)
        auto piece_of = [&](int j, int stream, int i, float2 (&v)[V / 2]) {
            const uint4 raw = live(j) ? *slot_of(stage, j, stream, i) : make_uint4(0u, 0u, 0u, 0u);
            unpack<T>(SHIFT ? masked(raw, mask[i]) : raw, v);
        };
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                float2 h[V / 2], dy[V / 2], w2[V / 2];
                piece_of(j, 1, i, h);
                piece_of(j, 2, i, dy);
                param_piece(2, i, column(i), w2);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    // (rstd behind the sum: outside the row the gradient is 0 and h - mean a number, but (0 - mean) rstd may be infinite)
                    const float2 u = __fmul2_rn(dy[e], __fadd2_rn(h[e], both(-mean2[j])));
                    if constexpr (kSums) {
                        sums[0][i][e] = __ffma2_rn(u, both(rstd2[j]), sums[0][i][e]);
                        sums[1][i][e] = __fadd2_rn(sums[1][i][e], dy[e]);
                    }
                    s0 = __ffma2_rn(dy[e], w2[e], s0);
                    s1 = __ffma2_rn(u, w2[e], s1);
                }
            }
            s[2 * j] = s0.x + s0.y;
            s[2 * j + 1] = s1.x + s1.y;
        }
        reduce(s, [&](float all) { return all * inv_C; });
        float2 by[R][ITEMS][V / 2];  // what goes into the first norm's gradient
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float2 t0 = both(0.0f), t1 = both(0.0f), tg = both(0.0f);
            const float m1 = s[2 * j], m2 = s[2 * j + 1] * rstd2[j] * rstd2[j];
            if constexpr (!kSums)
                if (threadIdx.x == 0 && live(j) && a.row_sums) {
                    a.row_sums[row0 + j * step] = m1;
                    a.row_sums[a.rows + row0 + j * step] = s[2 * j + 1] * rstd2[j];
                }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = column(i);
                float2 d[V / 2], h[V / 2], x[V / 2], n[V / 2], w[V / 2];
                piece_of(j, 1, i, h);
                piece_of(j, 2, i, d);
                param_piece(2, i, c, w);
#pragma unroll
                for (int e = 0; e < V / 2; ++e)
                    d[e] = __ffma2_rn(__fadd2_rn(h[e], both(-mean2[j])), both(-m2), __ffma2_rn(d[e], w[e], both(-m1)));
                piece_of(j, 3, i, h);
                piece_of(j, 0, i, x);
                param_piece(0, i, c, w);
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    d[e] = __ffma2_rn(d[e], both(rstd2[j]), h[e]);
                    x[e] = __fadd2_rn(x[e], both(-mean1[j]));  // (rstd behind the sums, as above)
                }
                if (live(j) && a.grad_residual) store_piece<T, SHIFT>(to_onto.of(j, i * apart), c, a.C, pack<T>(d));
                if constexpr (G != Gate::None) {
                    param_piece(1, i, c, n);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) n[e] = __fmul2_rn(d[e], __ffma2_rn(__fmul2_rn(x[e], both(rstd1[j])), w[e], n[e]));
                }
                if constexpr (G == Gate::All) {
                    if (live(j) && a.grad_gate) store_piece<T, SHIFT>(to_gate.of(j, i * apart), c, a.C, pack<T>(n));
                    float2 g[V / 2];
                    piece_of(j, 4, i, g);
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
                    if constexpr (kSums) {
                        sums[2][i][e] = __ffma2_rn(u, both(rstd1[j]), sums[2][i][e]);
                        sums[3][i][e] = __fadd2_rn(sums[3][i][e], d[e]);
                    }
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
    if constexpr (!kSums) return;
    if (!a.parts) return;
    float* part = a.parts + static_cast<long long>(blockIdx.x) * 4 * a.C;
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
                            make_float4(sums[k][kSums ? i : 0][e].x, sums[k][kSums ? i : 0][e].y, sums[k][kSums ? i : 0][e + 1].x, sums[k][kSums ? i : 0][e + 1].y);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (static_cast<unsigned>(c + e) < static_cast<unsigned>(a.C)) part[k * a.C + c + e] = at_of(sums[k][kSums ? i : 0], e);
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
                            for (int k = 0; k < 4; ++k) own[k * a.C + c] = at_of(sums[k][kSums ? i : 0], e) + (q ? own[k * a.C + c] : 0.0f);
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

// Blocks and rows under way: as many blocks per SM as registers allow, with what they may have of shared memory
struct RowShape {
    RowPlan p;
    int blocks, depth;
    size_t smem;
};
// (sums' slots and rows' numbers)
constexpr int kStaticBytes = (2 * SumOf<false>::kSlots + 5 * kNumberRows) * sizeof(float) + 256;
// extra: bytes of a block beside its rows
bool shape_of(const RowPlan& p, long long rows, int R, int streams, long long extra, int per_sm, const DeviceCtx* ctx, RowShape* s) {
    const long long row_bytes = static_cast<long long>(R) * streams * p.items * p.threads * 16;
    auto room = [&] { return ctx->max_smem_optin / per_sm - 1024 - kStaticBytes - extra; };
    s->p = p;
    s->depth = ring_depth(row_bytes, room());
    while (s->depth < 2 && per_sm > 1) {
        --per_sm;
        s->depth = ring_depth(row_bytes, room());
    }
    if (s->depth < 1) return false;
    const long long needed = (rows + p.rows_per_block() - 1) / p.rows_per_block();
    long long blocks = static_cast<long long>(per_sm) * ctx->sm_count;
    if (p.shift && !p.group) blocks = blocks / 8 * 8;
    if (needed < blocks) blocks = needed;  // (a block has one row at most, then, and it does not matter how far they are apart)
    const long long turns = (needed + R * blocks - 1) / (R * blocks);
    if (turns < s->depth) s->depth = static_cast<int>(turns);
    s->blocks = static_cast<int>(blocks);
    s->smem = static_cast<size_t>(s->depth * row_bytes + extra);
    return true;
}
// Calls f with a variant's numbers.  Blocks' rows: 16 elements per thread of 16 bits (the instructions around an element count: 16384 x 5120
// with 8 took 203 and 415 us), 8 of 32; 32 where that does not reach.
template <class T, class F>
int with_items(const RowPlan& p, F f) {
    constexpr int k8 = 8 / kPiece<T>, k16 = 16 / kPiece<T>, k32 = 32 / kPiece<T>, kBlock = sizeof(T) == 4 ? k8 : k16;
    using std::integral_constant;
    auto go = [&](auto items, auto group) { return p.shift ? f(items, group, std::true_type()) : f(items, group, std::false_type()); };
    if (p.group) return p.items == k8 ? go(integral_constant<int, k8>(), std::true_type()) : go(integral_constant<int, k16>(), std::true_type());
    return p.items == kBlock ? go(integral_constant<int, kBlock>(), std::false_type()) : go(integral_constant<int, k32>(), std::false_type());
}
template <class F>
int with_gate(Gate gate, F f) {
    switch (gate) {
        case Gate::None: return f(std::integral_constant<Gate, Gate::None>());
        case Gate::Row: return f(std::integral_constant<Gate, Gate::Row>());
        default: return f(std::integral_constant<Gate, Gate::All>());
    }
}
// Blocks of a kernel that an SM's registers hold, and the kernel's right to shared memory
template <auto KERNEL>
int resident_blocks(int threads, const DeviceCtx* ctx, int* per_sm) {
    static OncePerDevice once;
    const int r = once([&] { return allow_smem(KERNEL, ctx->max_smem_optin - kStaticBytes); });
    if (r != kOk) return r;
    static std::atomic<int> resident[64][33];
    std::atomic<int>& known = resident[ctx->device][threads / 32];
    *per_sm = known.load(std::memory_order_acquire);
    if (*per_sm == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, KERNEL, threads, 0) != cudaSuccess || *per_sm < 1) {
            cudaGetLastError();
            *per_sm = 1;
        }
        known.store(*per_sm, std::memory_order_release);
    }
    return kOk;
}

bool plan_forward(Gate gate, const SandwichArgs& a, int type, RowPlan* p) {
    const int size = size_of(type);
    const bool aligned = on16(a.x) && on16(a.residual) && on16(a.h) && on16(a.y) && (gate != Gate::All || on16(a.gate));
    const bool match = rows_match(size, a.C, a.pitch, aligned) && rows_match(size, a.C, a.pitch_residual, aligned) &&
                       (gate != Gate::All || rows_match(size, a.C, a.pitch_gate, aligned));
    const bool shift = rows_shift(size, a.C) || !on16(a.p.scale) || !on16(a.p.post_weight) || !on16(a.p.post_bias) || !on16(a.p.weight) ||
                       !on16(a.p.bias);
    return match && plan_elements(a.C, size, shift, false, p);
}
bool plan_backward(Gate gate, const SandwichGradArgs& a, int type, RowPlan* p) {
    const int size = size_of(type);
    const bool aligned = on16(a.x) && on16(a.h) && on16(a.grad_y) && on16(a.grad_h) && on16(a.grad_x) && on16(a.grad_residual) &&
                         (gate != Gate::All || (on16(a.gate) && on16(a.grad_gate)));
    const bool match = rows_match(size, a.C, a.pitch, aligned) && (gate != Gate::All || rows_match(size, a.C, a.pitch_gate, aligned));
    const bool shift = rows_shift(size, a.C) || !on16(a.p.scale) || !on16(a.p.post_weight) || !on16(a.p.post_bias) || !on16(a.p.weight);
    return match && plan_elements(a.C, size, shift, false, p);
}
// The backward kernel for these rows, with its shape: f(kernel, shape); kBadArgument where there is none
template <class F>
int with_backward(Gate gate, const SandwichGradArgs& a, int type, const DeviceCtx* ctx, F f) {
    RowPlan p;
    if (!plan_backward(gate, a, type, &p)) return kBadArgument;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return with_gate(gate, [&](auto g) {
            return with_items<T>(p, [&](auto items, auto group, auto shift) {
                constexpr Gate G = decltype(g)::value;
                constexpr int kItems = decltype(items)::value;
                constexpr bool kGroup = decltype(group)::value;
                constexpr auto kernel = sandwich_grad_registers_kernel<T, G, kItems, kGroup, decltype(shift)::value>;
                int per_sm;
                const int r = resident_blocks<kernel>(p.threads, ctx, &per_sm);
                if (r != kOk) return r;
                RowShape s;
                const long long params = kGroup || kItems * kPiece<T> > 16 ? 0 : 3LL * kItems * (kPiece<T> / 4) * p.threads * 16;
                if (!shape_of(p, a.rows, 1, kBackwardStreams<G>, params, per_sm, ctx, &s)) return static_cast<int>(kBadArgument);
                if constexpr (kGroup) {
                    const size_t columns = static_cast<size_t>(kGroupThreads / 32) * 4 * a.C * sizeof(float);
                    if (s.smem < columns) s.smem = columns;
                }
                return f(kernel, s, kItems * kPiece<T> <= 16);
            });
        });
    });
}

}  // namespace

bool sandwich_in_registers(Gate gate, const SandwichArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st, int* status) {
    RowPlan p;
    if (!plan_forward(gate, a, type, &p)) return false;
    bool fits = true;
    const int r = with_type(type, [&](auto t) {
        using T = decltype(t);
        return with_gate(gate, [&](auto g) {
            return with_items<T>(p, [&](auto items, auto group, auto shift) {
                constexpr Gate G = decltype(g)::value;
                constexpr int kItems = decltype(items)::value;
                constexpr bool kGroup = decltype(group)::value;
                constexpr auto kernel = sandwich_registers_kernel<T, G, kItems, kGroup, decltype(shift)::value>;
                int per_sm;
                const int r = resident_blocks<kernel>(p.threads, ctx, &per_sm);
                if (r != kOk) return r;
                RowShape s;
                fits = shape_of(p, a.rows, rows_forward(kItems * kPiece<T>, sizeof(T), kGroup, decltype(shift)::value), kForwardStreams<G>, 0, per_sm, ctx, &s);
                return fits ? launch_after(kernel, s.blocks, p.threads, s.smem, st, a, p.lanes, s.depth) : static_cast<int>(kOk);
            });
        });
    });
    if (fits) *status = r;
    return fits;
}

int sandwich_grad_in_registers(Gate gate, const SandwichGradArgs& a, int type, const DeviceCtx* ctx, bool sums, int* blocks) {
    int on_chip = kNothing;
    with_backward(gate, a, type, ctx, [&](auto, const RowShape& s, bool with_sums) {
        *blocks = s.blocks;
        on_chip = with_sums || !sums ? kRowsAndSums : kRows;
        return static_cast<int>(kOk);
    });
    return on_chip;
}

int launch_sandwich_grad_in_registers(Gate gate, const SandwichGradArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st) {
    return with_backward(gate, a, type, ctx, [&](auto kernel, const RowShape& s, bool) {
        return launch_after(kernel, s.blocks, s.p.threads, s.smem, st, a, s.p.lanes, s.depth);
    });
}

bool sandwich_runs(Gate gate, const SandwichGradArgs& a, int type) {
    RowPlan p;
    return plan_backward(gate, a, type, &p) && !rows_shift(size_of(type), a.C);
}

}  // namespace ldn
