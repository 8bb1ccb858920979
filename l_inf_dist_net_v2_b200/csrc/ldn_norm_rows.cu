// Layer norm forward (and rows as integers) with rows in registers: one read of a row, two sums over it (the mean, then the squares of
// what is left), one write.
//
// Bound by memory: what a call cannot do without is x and y once (joined: x, the residual, h and y).  So a block always has rows
// under way, into shared memory without registers, and takes several rows at a time, whose sums share their barriers: with one row
// that was loaded when the one before was done, a 16384 x 5120 bf16 norm took 104 us at 49 % of the copy rate, with rows under
// way 65 to 68 at 76 % (50000 rows: 190 us at 83 %; 16383 x 4097, cut rows: 76 us at 54 %; as integers 131 us at 23 %).  A thread keeps
// its columns' weight and bias from row to row (a block takes every gridDim-th row; where rows start anywhere in 16 bytes the grid is
// a multiple of eight, and rows that far apart start alike).  Rows of 5121 to 16384 have no registers for that and read them again
// (8192 x 8192 bf16: 84 us at 49 %; 13104 x 5121, cut rows: 203 at 20 %).
#include "ldn_norm.cuh"
#include "ldn_rows.cuh"

namespace ldn {
namespace {

// Rows that a block takes at a time
__host__ __device__ constexpr int rows_at_once(Form f, int elements, bool group) {
    return group || elements > 16 || f == Form::Quantised ? 1 : elements > 8 || f == Form::Joined ? 2 : 4;
}
template <Form F>
constexpr int kStreams = F == Form::Joined ? 2 : 1;

// The integers of a piece, whose columns start at c0: words of four where memory allows, as pieces that are cut do not start at
// multiples of four bytes of the integers' row: the last `ahead` bytes of a word come from the next lane's piece.
template <int V, bool SHIFT>
__device__ __forceinline__ void store_integers(signed char* to, int c0, int C, const unsigned (&word)[V / 4], int lane_in_warp, int lanes) {
    if (!SHIFT) {  // (rows start at multiples of 16 bytes then)
        if (c0 < C) {
            if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[1]);
            else *reinterpret_cast<unsigned*>(to) = word[0];
        }
        return;
    }
    const unsigned next = __shfl_down_sync(0xffffffffu, word[0], 1);
    const int ahead = (4 - static_cast<int>(reinterpret_cast<uintptr_t>(to) & 3u)) & 3;
    const bool last = lane_in_warp == (lanes < 32 ? lanes : 32) - 1, begins = lane_in_warp == 0;
    if (c0 >= 0 && c0 + V + 4 <= C && !last) {
        unsigned w[V / 4 + 1];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) w[i] = word[i];
        w[V / 4] = next;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) *reinterpret_cast<unsigned*>(to + ahead + 4 * i) = __funnelshift_r(w[i], w[i + 1], 8 * ahead);
        if (!begins && c0 >= V) return;  // (its first bytes are the lane's in front)
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < ahead) to[e] = static_cast<signed char>(word[0] >> 8 * e);
    } else {
        // (those that the lane in front has stored are stored again: the same bytes)
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(C)) to[e] = static_cast<signed char>(word[e / 4] >> 8 * (e % 4));
    }
}

template <class T, Form F, int ITEMS, bool GROUP, bool SHIFT>
__global__ void __launch_bounds__(GROUP ? kGroupThreads : threads_of(ITEMS * kPiece<T>), !GROUP && ITEMS * kPiece<T> == 16 ? (F == Form::Quantised ? 4 : 2) : 1)
norm_registers_kernel(NormArgs a, int lanes, int depth) {
    if constexpr (F == Form::Quantised) {  // (what comes behind may read what was there before this kernel)
        stream_order_wait();
        stream_order_release();
    } else {
        stream_order_begin();
    }
    constexpr int V = kPiece<T>, S = kStreams<F>, R = rows_at_once(F, ITEMS * V, GROUP);
    constexpr bool kParams = F != Form::Quantised, kKeep = kParams && ITEMS * V <= 16;
    __shared__ float slots[2 * RowSum::kSlots];
    extern __shared__ uint4 ring[];  // [depth][row][stream][item][thread]
    RowSum reduce{lanes, slots, 0};
    Generator gen;
    if constexpr (F == Form::Joined) gen = generator_of(a.drop);
    const int lane = GROUP ? threadIdx.x & (lanes - 1) : threadIdx.x;
    const int per_block = GROUP ? kGroupThreads / lanes : 1;
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    const long long mine = static_cast<long long>(blockIdx.x) * per_block + (GROUP ? threadIdx.x / lanes : 0);
    const float inv_C = 1.0f / a.C;
    // (the same for all rows of this thread)
    const int shift = SHIFT ? shift_of(static_cast<const T*>(a.x) + (mine < a.rows ? mine : 0) * a.pitch) : 0;
    auto column = [&](int i) { return (lane + i * lanes) * V - shift; };
    float2 w[ITEMS][V / 2], b[ITEMS][V / 2];
    uint4 mask[ITEMS];
    int bytes[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        mask[i] = mask_of<T, SHIFT>(column(i), a.C);
        bytes[i] = piece_bytes<T>(column(i), a.C);
        if constexpr (kKeep) {
            load_params<T, SHIFT>(a.weight, a.wide, column(i), a.C, 1.0f, w[i]);
            load_params<T, SHIFT>(a.bias, a.wide, column(i), a.C, 0.0f, b[i]);
        }
    }
    // this thread's rows, and where their pieces are: those to be fetched, and those to be made
    const int c0 = column(0), apart = lanes * V;
    int to_fetch = mine < a.rows ? static_cast<int>((a.rows - mine + step - 1) / step) : 0, to_make = to_fetch;
    Walk<const T> from_x(a.x, a.pitch, mine, step, c0), from_onto(a.residual, a.pitch_residual, mine, step, c0);
    Walk<T> to_h(a.h, a.C, mine, step, c0), to_y(a.y, a.C, mine, step, c0);
    Walk<signed char> to_q(a.q, a.pitch_q, mine, step, c0);
    long long row0 = mine, index = mine * a.C + c0;
    uint4* own = ring + threadIdx.x;
    auto slot_of = [&](int stage, int j, int stream, int i) { return own + (((stage * R + j) * S + stream) * ITEMS + i) * blockDim.x; };
    auto fetch = [&](int stage) {
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (j < to_fetch) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    copy_piece<T, SHIFT>(slot_of(stage, j, 0, i), from_x.of(j, i * apart), column(i), bytes[i], a.x);
                    if constexpr (S == 2)
                        copy_piece<T, SHIFT>(slot_of(stage, j, 1, i), from_onto.of(j, i * apart), column(i), bytes[i], a.residual);
                }
            }
        copies_commit();
        to_fetch -= R;
        from_x.on(R);
        if (S == 2) from_onto.on(R);
    };
    for (int d = 0; d < depth * R * S; ++d)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (!bytes[i]) own[(d * ITEMS + i) * blockDim.x] = make_uint4(0u, 0u, 0u, 0u);
    for (int d = 0; d < depth; ++d) fetch(d);
    int stage = 0;
    // (a warp's groups take part in its shuffles whether they have a row or not: as many turns as the block's first has)
    const long long block_first = static_cast<long long>(blockIdx.x) * per_block;
    const int turns = block_first < a.rows ? static_cast<int>((a.rows - block_first + R * step - 1) / (R * step)) : 0;
    for (int turn = 0; turn < turns; ++turn) {
        auto live = [&](int j) { return j < to_make; };
        copies_wait(depth);
        float2 v[R][ITEMS][V / 2];
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = column(i);
                uint4 raw = live(j) ? *slot_of(stage, j, 0, i) : make_uint4(0u, 0u, 0u, 0u);
                if constexpr (F == Form::Joined) {
                    if (live(j)) {
                        float2 r[V / 2];
                        unpack<T>(raw, v[j][i]);
                        unpack<T>(*slot_of(stage, j, 1, i), r);
                        drop_piece(a.drop, gen, index + j * step * a.C + i * apart, v[j][i]);  // (pieces start at multiples of four elements)
#pragma unroll
                        for (int e = 0; e < V / 2; ++e) v[j][i][e] = __fadd2_rn(r[e], v[j][i][e]);
                        raw = pack<T>(v[j][i]);
                        store_piece<T, SHIFT>(to_h.of(j, i * apart), c, a.C, raw);
                    }
                    if (!SHIFT && c >= a.C) raw = make_uint4(0u, 0u, 0u, 0u);
                }
                unpack<T>(SHIFT ? masked(raw, mask[i]) : raw, v[j][i]);
            }
        fetch(stage);
        stage = stage + 1 == depth ? 0 : stage + 1;
        if constexpr (kParams) {
            float s[R], mean[R];
#pragma unroll
            for (int j = 0; j < R; ++j) {
                float2 sum = both(0.0f);
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) sum = __fadd2_rn(sum, v[j][i][e]);
                s[j] = sum.x + sum.y;
            }
            reduce.template sum<GROUP>(s, [&](float all) { return all * inv_C; });
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
            reduce.template sum<GROUP>(s, [&](float all) { return 1.0f / sqrtf(all * inv_C + a.eps); });
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (lane == 0 && a.mean && live(j)) {
                    a.mean[row0 + j * step] = mean[j];
                    a.rstd[row0 + j * step] = s[j];
                }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = column(i);
                if constexpr (!kKeep) {
                    load_params<T, SHIFT>(a.weight, a.wide, c, a.C, 1.0f, w[i]);
                    load_params<T, SHIFT>(a.bias, a.wide, c, a.C, 0.0f, b[i]);
                }
#pragma unroll
                for (int j = 0; j < R; ++j) {
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) v[j][i][e] = __ffma2_rn(__fmul2_rn(v[j][i][e], both(s[j])), w[i][e], b[i][e]);
                    if constexpr (F != Form::Integers)
                        if (live(j)) store_piece<T, SHIFT>(to_y.of(j, i * apart), c, a.C, pack<T>(v[j][i]));
                }
            }
        }
        if constexpr (F == Form::Integers || F == Form::Quantised) {
            float top[R];
#pragma unroll
            for (int j = 0; j < R; ++j) {
                top[j] = 0.0f;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    if constexpr (F == Form::Integers) only_row<SHIFT>(column(i), a.C, v[j][i]);  // (a bias of nothing may be there)
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) top[j] = larger(top[j], v[j][i][e]);
                }
            }
            reduce.template largest<GROUP>(top, [](float all) { return step_of(__float_as_uint(all)); });
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const float size = top[j], inverse = 1.0f / size;
                if (lane == 0 && live(j)) a.scale[row0 + j * step] = size;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    unsigned word[V / 4];
#pragma unroll
                    for (int e = 0; e < V / 4; ++e) word[e] = steps4(v[j][i][2 * e], v[j][i][2 * e + 1], inverse);
                    store_integers<V, SHIFT>(to_q.of(j, i * apart), column(i), live(j) ? a.C : 0, word, GROUP ? lane : threadIdx.x & 31,
                                             lanes);
                }
            }
        }
        to_make -= R;
        row0 += R * step;
        if constexpr (F == Form::Joined) {
            to_h.on(R);
            index += R * step * a.C;
        }
        if constexpr (F == Form::Plain || F == Form::Joined) to_y.on(R);
        else to_q.on(R);
    }
}

template <class T, Form F, int ITEMS, bool GROUP, bool SHIFT>
int launch(const NormArgs& a, const RowPlan& p, const DeviceCtx* ctx, cudaStream_t st) {
    constexpr auto kernel = norm_registers_kernel<T, F, ITEMS, GROUP, SHIFT>;
    static OncePerDevice once;
    const int most_smem = ctx->max_smem_optin - 2560;
    int r = once([&] { return allow_smem(kernel, most_smem); });
    if (r != kOk) return r;
    // as many blocks as registers allow, with what they may have of shared memory
    static std::atomic<int> resident[64][33];
    std::atomic<int>& known = resident[ctx->device][p.threads / 32];
    int per_sm = known.load(std::memory_order_acquire);
    if (per_sm == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, p.threads, 0) != cudaSuccess || per_sm < 1) {
            cudaGetLastError();
            per_sm = 1;
        }
        known.store(per_sm, std::memory_order_release);
    }
    constexpr int R = rows_at_once(F, ITEMS * kPiece<T>, GROUP);
    const long long row_bytes = static_cast<long long>(R) * kStreams<F> * ITEMS * p.threads * 16;
    int depth = ring_depth(row_bytes, most_smem / per_sm - 1024);
    while (depth < 2 && per_sm > 1) depth = ring_depth(row_bytes, most_smem / --per_sm - 1024);
    if (depth < 1) depth = 1;  // (a row of 16384 in 32 bits and its residual: 128 KB)
    const long long needed = (a.rows + p.rows_per_block() - 1) / p.rows_per_block();
    long long blocks = static_cast<long long>(per_sm) * ctx->sm_count;
    if (p.shift && !p.group) blocks = blocks / 8 * 8;
    if (needed < blocks) blocks = needed;  // (a block has one row at most, then, and it does not matter how far they are apart)
    const long long turns = (needed + R * blocks - 1) / (R * blocks);
    if (turns < depth) depth = static_cast<int>(turns);
    return launch_after(kernel, static_cast<unsigned>(blocks), p.threads, depth * row_bytes, st, a, p.lanes, depth);
}
template <class T, Form F>
int launch(const NormArgs& a, const RowPlan& p, const DeviceCtx* ctx, cudaStream_t st) {
    constexpr int k8 = 8 / kPiece<T>, k16 = 16 / kPiece<T>, k32 = 32 / kPiece<T>;
    constexpr int kBlock = F == Form::Joined || sizeof(T) == 4 ? k8 : k16;  // (as plan_elements has it)
    if (p.group && p.items == k8) return p.shift ? launch<T, F, k8, true, true>(a, p, ctx, st) : launch<T, F, k8, true, false>(a, p, ctx, st);
    if (p.group) return p.shift ? launch<T, F, k16, true, true>(a, p, ctx, st) : launch<T, F, k16, true, false>(a, p, ctx, st);
    if (p.items == kBlock) return p.shift ? launch<T, F, kBlock, false, true>(a, p, ctx, st) : launch<T, F, kBlock, false, false>(a, p, ctx, st);
    return p.shift ? launch<T, F, k32, false, true>(a, p, ctx, st) : launch<T, F, k32, false, false>(a, p, ctx, st);
}

}  // namespace

bool norm_in_registers(Form form, const NormArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st, int* status) {
    const int size = size_of(type);
    bool aligned = on16(a.x) && on16(a.y) && on16(a.h) && on16(a.residual);  // (the ones that the form has not are null)
    bool match = rows_match(size, a.C, a.pitch, aligned);
    if (form == Form::Joined) match = match && rows_match(size, a.C, a.pitch_residual, aligned);
    bool shift = rows_shift(size, a.C) || !on16(a.weight) || !on16(a.bias);
    if (form == Form::Integers || form == Form::Quantised) {
        // nothing has to match x but the integers, which are put together where they do not
        match = (reinterpret_cast<uintptr_t>(a.x) & (size - 1)) == 0;
        shift = shift || !on16(a.x) || a.pitch * size % 16 != 0 || !on16(a.q) || a.pitch_q % 16 != 0;
    }
    RowPlan p;
    if (!match || !plan_elements(a.C, size, shift, form == Form::Joined, &p)) return false;
    *status = with_type(type, [&](auto t) {
        using T = decltype(t);
        switch (form) {
            case Form::Plain: return launch<T, Form::Plain>(a, p, ctx, st);
            case Form::Joined: return launch<T, Form::Joined>(a, p, ctx, st);
            case Form::Integers: return launch<T, Form::Integers>(a, p, ctx, st);
            default: return launch<T, Form::Quantised>(a, p, ctx, st);
        }
    });
    return true;
}

}  // namespace ldn
