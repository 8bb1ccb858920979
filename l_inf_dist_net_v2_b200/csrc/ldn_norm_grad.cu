// Layer norm's gradient with the row in registers: one read of x and of the incoming gradients, both sums over a row at once, and
// the column sums for the weight and the bias carried in the threads that have those columns, from row to row.
//
// A block takes every gridDim-th row, so its threads' columns stay (rows that start anywhere in 16 bytes: the grid is a multiple of
// eight, and rows that far apart start alike).  The next row is under way while this one is summed.  Bound by memory: x, the incoming
// and the outgoing gradients once.
#include "ldn_norm.cuh"
#include "ldn_rows.cuh"

namespace ldn {
namespace {

// 16 elements per thread, whose 32 column sums stay in registers: rows of up to 8192
constexpr int kMostThreads = 512;
template <class T>
constexpr int kMostItems = 16 / kPiece<T>;

template <class T, bool JOINED, int ITEMS, bool GROUP, bool SHIFT>
__global__ void __launch_bounds__(GROUP ? kGroupThreads : kMostThreads) norm_grad_registers_kernel(NormGradArgs a, int lanes) {
    stream_order_begin();
    constexpr int V = kPiece<T>;
    __shared__ float slots[128];
    extern __shared__ float columns[];  // groups: [warp][2][C]
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
    float sum_w[ITEMS][V], sum_b[ITEMS][V];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) sum_w[i][e] = sum_b[i][e] = 0.0f;

    uint4 next_x[ITEMS], next_g[ITEMS];
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto fetch = [&](long long row) {
        const bool live = row < a.rows;
        const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.pitch;
        const T* g = static_cast<const T*>(a.grad_y) + (live ? row : 0) * a.C;
        const int C = live ? a.C : 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            next_x[i] = load_piece<T, SHIFT>(x, (lane + i * lanes) * V - shift, C);
            next_g[i] = load_piece<T, SHIFT>(g, (lane + i * lanes) * V - shift, C);
        }
        next_mean = live ? a.mean[row] : 0.0f;
        next_rstd = live ? a.rstd[row] : 0.0f;
    };
    fetch(mine);
    // (a warp's groups take part in its shuffles whether they have a row or not)
    for (long long first = static_cast<long long>(blockIdx.x) * per_block; first < a.rows; first += step) {
        const long long row = GROUP ? first + threadIdx.x / lanes : first;
        const bool live = !GROUP || row < a.rows;
        const long long at = (live ? row : 0) * a.C;
        const int C = live ? a.C : 0;
        uint4 x[ITEMS], g[ITEMS], more[ITEMS];
        const float mean = next_mean, rstd = next_rstd;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            x[i] = next_x[i];
            g[i] = next_g[i];
        }
        if constexpr (JOINED) {
            if (a.grad_h)
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
                    more[i] = load_piece<T, SHIFT>(static_cast<const T*>(a.grad_h) + at, (lane + i * lanes) * V - shift, C);
        }
        fetch(row + step);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c0 = (lane + i * lanes) * V - shift;
            float vx[V], vg[V], w[V];
            unpack<T>(x[i], vx);
            unpack<T>(g[i], vg);
            load_params<T, SHIFT>(a.weight, a.wide, c0, C, 1.0f, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {  // (outside the row the gradient is 0)
                const float z = (vx[e] - mean) * rstd;
                sum_w[i][e] = fmaf(vg[e], z, sum_w[i][e]);
                sum_b[i][e] += vg[e];
                const float p = vg[e] * w[e];
                s[0] += p;
                s[1] = fmaf(p, z, s[1]);
            }
        }
        reduce.template sum<2, GROUP>(s);
        const float m1 = s[0] * inv_C, m2 = s[1] * inv_C;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c0 = (lane + i * lanes) * V - shift;
            float vx[V], vg[V], w[V];
            unpack<T>(x[i], vx);
            unpack<T>(g[i], vg);
            load_params<T, SHIFT>(a.weight, a.wide, c0, C, 1.0f, w);
#pragma unroll
            for (int e = 0; e < V; ++e) vg[e] = rstd * (vg[e] * w[e] - m1 - (vx[e] - mean) * rstd * m2);
            if constexpr (JOINED) {
                if (a.grad_h) {
                    float vh[V];
                    unpack<T>(more[i], vh);
#pragma unroll
                    for (int e = 0; e < V; ++e) vg[e] += vh[e];
                }
                if (a.grad_residual) store_piece<T, SHIFT>(static_cast<T*>(a.grad_residual) + at, c0, C, pack<T>(vg));
                if (a.grad_x)
#pragma unroll
                    for (int e = 0; e < V; e += 4) {  // (pieces start at multiples of four elements of the whole tensor)
                        const uint4 r = random_words(gen, static_cast<unsigned long long>(at + c0 + e) >> 2);
                        vg[e] = dropped(a.drop, r.x, vg[e]);
                        vg[e + 1] = dropped(a.drop, r.y, vg[e + 1]);
                        vg[e + 2] = dropped(a.drop, r.z, vg[e + 2]);
                        vg[e + 3] = dropped(a.drop, r.w, vg[e + 3]);
                    }
            }
            if (a.grad_x) store_piece<T, SHIFT>(static_cast<T*>(a.grad_x) + at, c0, C, pack<T>(vg));
        }
    }
    if (!a.parts) return;
    float* part = a.parts + static_cast<long long>(blockIdx.x) * 2 * a.C;
    if constexpr (!GROUP) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c0 = (lane + i * lanes) * V - shift;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(a.C)) {
                    part[c0 + e] = sum_w[i][e];
                    part[a.C + c0 + e] = sum_b[i][e];
                }
        }
    } else {
        // a warp's groups add to its columns in turn, then the warps' are added up
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
                            own[c0 + e] = sum_w[i][e] + (k ? own[c0 + e] : 0.0f);
                            own[a.C + c0 + e] = sum_b[i][e] + (k ? own[a.C + c0 + e] : 0.0f);
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

int smem_of(const RowPlan& p, int C) { return p.group ? kGroupThreads / 32 * 2 * C * static_cast<int>(sizeof(float)) : 0; }

template <class T, bool JOINED, int ITEMS, bool GROUP, bool SHIFT>
int run(const NormGradArgs& a, const RowPlan& p, const DeviceCtx* ctx, cudaStream_t st, int blocks) {
    // groups keep up to 1024 columns' sums per warp
    constexpr int kMostSmem = kGroupThreads / 32 * 2 * 32 * 16 * static_cast<int>(sizeof(float));
    static OncePerDevice once;
    if (GROUP) {
        const int r = once([] { return allow_smem(norm_grad_registers_kernel<T, JOINED, ITEMS, GROUP, SHIFT>, kMostSmem); });
        if (r != kOk) return r;
    }
    return launch_after(norm_grad_registers_kernel<T, JOINED, ITEMS, GROUP, SHIFT>, blocks, p.threads, smem_of(p, a.C), st, a, p.lanes);
}
template <class T, bool JOINED, int ITEMS>
int run(const NormGradArgs& a, const RowPlan& p, const DeviceCtx* ctx, cudaStream_t st, int blocks) {
    if (p.group)
        return p.shift ? run<T, JOINED, ITEMS, true, true>(a, p, ctx, st, blocks) : run<T, JOINED, ITEMS, true, false>(a, p, ctx, st, blocks);
    return p.shift ? run<T, JOINED, ITEMS, false, true>(a, p, ctx, st, blocks) : run<T, JOINED, ITEMS, false, false>(a, p, ctx, st, blocks);
}

bool plan_of(bool joined, const NormGradArgs& a, int type, RowPlan* p) {
    const int size = size_of(type);
    const bool aligned = on16(a.x) && on16(a.grad_y) && on16(a.grad_h) && on16(a.grad_x) && on16(a.grad_residual);
    const bool shift = rows_shift(size, a.C) || !on16(a.weight);
    return rows_match(size, a.C, a.pitch, aligned) && plan_rows(a.C, 16 / size, shift, size, kMostThreads, 1, p);
}
int blocks_of(const RowPlan& p, const NormGradArgs& a, const DeviceCtx* ctx) {
    const long long needed = (a.rows + p.rows_per_block() - 1) / p.rows_per_block();
    const int per_sm = p.threads <= 192 ? 4 : p.threads <= 256 ? 3 : p.threads <= 384 ? 2 : 1;
    long long most = static_cast<long long>(per_sm) * ctx->sm_count;
    if (p.shift && !p.group) {
        most = most / 8 * 8;
        return static_cast<int>(needed < most ? (needed + 7) / 8 * 8 : most);  // (blocks without rows give parts of zeros)
    }
    return static_cast<int>(needed < most ? needed : most);
}

}  // namespace

bool norm_grad_in_registers(bool joined, const NormGradArgs& a, int type, const DeviceCtx* ctx, int* blocks) {
    RowPlan p;
    if (!plan_of(joined, a, type, &p)) return false;
    *blocks = blocks_of(p, a, ctx);
    return true;
}

int launch_norm_grad_in_registers(bool joined, const NormGradArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st) {
    RowPlan p;
    if (!plan_of(joined, a, type, &p)) return kBadArgument;
    const int blocks = blocks_of(p, a, ctx);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        auto by_items = [&](auto j) {
            constexpr bool J = decltype(j)::value;
            switch (p.items) {
                case 1: return run<T, J, 1>(a, p, ctx, st, blocks);
                case 2: return run<T, J, 2>(a, p, ctx, st, blocks);
                default: return run<T, J, kMostItems<T>>(a, p, ctx, st, blocks);
            }
        };
        return joined ? by_items(std::true_type()) : by_items(std::false_type());
    });
}

}  // namespace ldn
