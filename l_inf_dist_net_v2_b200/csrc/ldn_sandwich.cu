// The residual stream between two norms: kernels for rows of any length, alignment and pitch, the fold of the column sums, and the entry
// points.  Statistics are those of two passes, in 32 bits; h is rounded before it is normalised, so the backward pass sees what the
// forward pass used.
#include "ldn_sandwich.cuh"

namespace ldn {
namespace {

constexpr int kRowThreads = 256;

// A block per row, an element per thread and step; a row is read again for every pass (9999 x 1001 f16: 129 us, 35 with rows in registers).
template <class T, Gate G>
__global__ void __launch_bounds__(kRowThreads) sandwich_rows_kernel(const __grid_constant__ SandwichArgs a) {
    stream_order_begin();
    __shared__ float slots[kRowThreads / 32];
    const T* gates = static_cast<const T*>(a.gate);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.pitch;
        T* h = static_cast<T*>(a.h) + row * a.C;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) sum += to_float(x[c]);
        const float mean1 = block_sum(sum, slots) / a.C;
        sum = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            const float d = to_float(x[c]) - mean1;
            sum += d * d;
        }
        const float rstd1 = 1.0f / sqrtf(block_sum(sum, slots) / a.C + a.eps);
        const float row_gate = G == Gate::Row ? to_float(gates[row]) : 1.0f;
        sum = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            const float n = (to_float(x[c]) - mean1) * rstd1 * param_or<T>(a.p.post_weight, a.p.wide, c, 1.0f) +
                            param_or<T>(a.p.post_bias, a.p.wide, c, 0.0f);
            const float gate = G == Gate::All ? to_float(gates[row * a.pitch_gate + c]) : row_gate;
            const T v = from_float<T>(to_float(static_cast<const T*>(a.residual)[row * a.pitch_residual + c]) +
                                      gate * (param_or<T>(a.p.scale, a.p.wide, c, 1.0f) * n));
            h[c] = v;  // (a thread reads back what it wrote)
            sum += to_float(v);
        }
        const float mean2 = block_sum(sum, slots) / a.C;
        sum = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            const float d = to_float(h[c]) - mean2;
            sum += d * d;
        }
        const float rstd2 = 1.0f / sqrtf(block_sum(sum, slots) / a.C + a.eps);
        for (int c = threadIdx.x; c < a.C; c += kRowThreads)
            static_cast<T*>(a.y)[row * a.C + c] = from_float<T>((to_float(h[c]) - mean2) * rstd2 * param_or<T>(a.p.weight, a.p.wide, c, 1.0f) +
                                                                param_or<T>(a.p.bias, a.p.wide, c, 0.0f));
        if (threadIdx.x == 0 && a.stats) {
            a.stats[row] = mean1;
            a.stats[a.rows + row] = rstd1;
            a.stats[2 * a.rows + row] = mean2;
            a.stats[3 * a.rows + row] = rstd2;
        }
    }
}

// The gradient of h at an element, given the row's two means
template <class T>
__device__ __forceinline__ float stream_gradient(const SandwichGradArgs& a, long long at, int c, float z2, float rstd2, float m1, float m2) {
    float d = a.grad_h ? to_float(static_cast<const T*>(a.grad_h)[at]) : 0.0f;
    if (a.grad_y) d += rstd2 * (to_float(static_cast<const T*>(a.grad_y)[at]) * param_or<T>(a.p.weight, a.p.wide, c, 1.0f) - m1 - z2 * m2);
    return d;
}

template <class T, Gate G>
__global__ void __launch_bounds__(kRowThreads) sandwich_grad_rows_kernel(const __grid_constant__ SandwichGradArgs a) {
    stream_order_begin();
    __shared__ float slots[kRowThreads / 32];
    const T* gates = static_cast<const T*>(a.gate);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T*>(a.x) + row * a.pitch, *h = static_cast<const T*>(a.h) + row * a.C;
        const long long at = row * a.C;
        const float mean1 = a.stats[row], rstd1 = a.stats[a.rows + row], mean2 = a.stats[2 * a.rows + row], rstd2 = a.stats[3 * a.rows + row];
        float m1 = 0.0f, m2 = 0.0f;
        if (a.grad_y)
            for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
                const float g = to_float(static_cast<const T*>(a.grad_y)[at + c]) * param_or<T>(a.p.weight, a.p.wide, c, 1.0f);
                m1 += g;
                m2 += g * ((to_float(h[c]) - mean2) * rstd2);
            }
        m1 = block_sum(m1, slots) / a.C;
        m2 = block_sum(m2, slots) / a.C;
        if (threadIdx.x == 0) {
            a.row_sums[row] = m1;
            a.row_sums[a.rows + row] = m2;
        }
        const float row_gate = G == Gate::Row ? to_float(gates[row]) : 1.0f;
        float s1 = 0.0f, s2 = 0.0f, sg = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            const float d = stream_gradient<T>(a, at + c, c, (to_float(h[c]) - mean2) * rstd2, rstd2, m1, m2);
            if (a.grad_residual) static_cast<T*>(a.grad_residual)[at + c] = from_float<T>(d);
            const float scale = param_or<T>(a.p.scale, a.p.wide, c, 1.0f), w1 = param_or<T>(a.p.post_weight, a.p.wide, c, 1.0f);
            const float z1 = (to_float(x[c]) - mean1) * rstd1, by_scale = d * scale;
            const float by_gate = by_scale * (z1 * w1 + param_or<T>(a.p.post_bias, a.p.wide, c, 0.0f));
            if (G == Gate::All && a.grad_gate) static_cast<T*>(a.grad_gate)[at + c] = from_float<T>(by_gate);
            const float b = by_scale * w1 * (G == Gate::All ? to_float(gates[row * a.pitch_gate + c]) : row_gate);
            s1 += b;
            s2 += b * z1;
            sg += by_gate;
        }
        s1 = block_sum(s1, slots) / a.C;
        s2 = block_sum(s2, slots) / a.C;
        if (G == Gate::Row && a.grad_gate) {
            sg = block_sum(sg, slots);
            if (threadIdx.x == 0) static_cast<T*>(a.grad_gate)[row] = from_float<T>(sg);
        }
        if (!a.grad_x) continue;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            const float d = stream_gradient<T>(a, at + c, c, (to_float(h[c]) - mean2) * rstd2, rstd2, m1, m2);
            const float z1 = (to_float(x[c]) - mean1) * rstd1;
            const float b = d * param_or<T>(a.p.scale, a.p.wide, c, 1.0f) * param_or<T>(a.p.post_weight, a.p.wide, c, 1.0f) *
                            (G == Gate::All ? to_float(gates[row * a.pitch_gate + c]) : row_gate);
            static_cast<T*>(a.grad_x)[at + c] = from_float<T>(rstd1 * (b - s1 - z1 * s2));
        }
    }
}

constexpr int kColumns = 32, kColumnLanes = 8;

// Column sums over a block of rows, behind the rows' means: a thread has a column and every eighth row, four of them under way.
template <class T, Gate G>
__global__ void __launch_bounds__(kColumns * kColumnLanes) sandwich_grad_columns_kernel(const __grid_constant__ SandwichGradArgs a) {
    stream_order_begin();
    constexpr int kAhead = 4;
    __shared__ float sums[4][kColumnLanes][kColumns];
    const int lane = threadIdx.x % kColumns, part = threadIdx.x / kColumns, c = blockIdx.x * kColumns + lane;
    const long long first = a.rows * blockIdx.y / gridDim.y, last = a.rows * (blockIdx.y + 1) / gridDim.y;
    const T* gates = static_cast<const T*>(a.gate);
    float s[4] = {};
    if (c < a.C)
        for (long long row0 = first + part; row0 < last; row0 += kAhead * kColumnLanes) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const long long row = row0 + u * kColumnLanes, at = row * a.C + c;
                if (row >= last) continue;
                const float rstd2 = a.stats[3 * a.rows + row];
                const float z2 = a.grad_y ? (to_float(static_cast<const T*>(a.h)[at]) - a.stats[2 * a.rows + row]) * rstd2 : 0.0f;
                const float z1 = (to_float(static_cast<const T*>(a.x)[row * a.pitch + c]) - a.stats[row]) * a.stats[a.rows + row];
                const float g = a.grad_y ? to_float(static_cast<const T*>(a.grad_y)[at]) : 0.0f;
                float d = stream_gradient<T>(a, at, c, z2, rstd2, a.row_sums[row], a.row_sums[a.rows + row]);
                if (G == Gate::Row) d *= to_float(gates[row]);
                if (G == Gate::All) d *= to_float(gates[row * a.pitch_gate + c]);
                s[0] += g * z2;
                s[1] += g;
                s[2] += d * z1;
                s[3] += d;
            }
        }
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[k][part][lane] = s[k];
    __syncthreads();
    if (part < 4 && c < a.C) {
        float all = 0.0f;
        for (int i = 0; i < kColumnLanes; ++i) all += sums[part][i][lane];
        a.parts[(static_cast<long long>(blockIdx.y) * 4 + part) * a.C + c] = all;
    }
}

struct FoldArgs {
    const float* parts;
    int count, C;
    SandwichParams p;
    void *scale, *post_weight, *post_bias, *weight, *bias;  // gradients; any may be null
};
// The parts in order: a thread has a column of one of the four sums and every fourth part, eight of them under way.
constexpr int kFoldLanes = 4, kFoldAhead = 8;
template <class T>
__global__ void __launch_bounds__(kColumns * 4 * kFoldLanes) sandwich_fold_kernel(const __grid_constant__ FoldArgs a) {
    stream_order_begin();
    __shared__ float sums[4][kFoldLanes][kColumns];
    const int lane = threadIdx.x % kColumns, k = threadIdx.x / kColumns % 4, part = threadIdx.x / (4 * kColumns), c = blockIdx.x * kColumns + lane;
    float s = 0.0f;
    if (c < a.C)
        for (int i = part; i < a.count; i += kFoldAhead * kFoldLanes) {
            float v[kFoldAhead];
#pragma unroll
            for (int u = 0; u < kFoldAhead; ++u) {
                const int j = i + u * kFoldLanes;
                v[u] = j < a.count ? a.parts[(4LL * j + k) * a.C + c] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < kFoldAhead; ++u) s += v[u];
        }
    sums[k][part][lane] = s;
    __syncthreads();
    if (threadIdx.x >= kColumns || c >= a.C) return;
    float all[4] = {};
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < kFoldLanes; ++i) all[q] += sums[q][i][lane];
    const float scale = param_or<T>(a.p.scale, a.p.wide, c, 1.0f);
    if (a.weight) set_param<T>(a.weight, a.p.wide, c, all[0]);
    if (a.bias) set_param<T>(a.bias, a.p.wide, c, all[1]);
    if (a.post_weight) set_param<T>(a.post_weight, a.p.wide, c, scale * all[2]);
    if (a.post_bias) set_param<T>(a.post_bias, a.p.wide, c, scale * all[3]);
    if (a.scale)
        set_param<T>(a.scale, a.p.wide, c,
                     param_or<T>(a.p.post_weight, a.p.wide, c, 1.0f) * all[2] + param_or<T>(a.p.post_bias, a.p.wide, c, 0.0f) * all[3]);
}

template <class F>
int with_gate(Gate gate, F f) {
    switch (gate) {
        case Gate::None: return f(std::integral_constant<Gate, Gate::None>());
        case Gate::Row: return f(std::integral_constant<Gate, Gate::Row>());
        default: return f(std::integral_constant<Gate, Gate::All>());
    }
}
bool sandwich_fits(long long rows, int C, int type, int param_type, int gate) {
    return rows >= 0 && row_fits(C) && known_type(type) && (param_type == LDN_F32 || param_type == type) && gate >= LDN_GATE_NONE &&
           gate <= LDN_GATE_ALL;
}

}  // namespace
}  // namespace ldn

using namespace ldn;

extern "C" LDN_API int ldn_sandwich_norm(const void* x, long long pitch, const void* residual, long long pitch_residual, const void* gate,
                                         long long pitch_gate, int gate_kind, long long rows, int C, int type, const void* scale,
                                         const void* post_weight, const void* post_bias, const void* weight, const void* bias, int param_type,
                                         float eps, void* h, void* y, float* stats, ldn_stream_t stream) {
    if (!sandwich_fits(rows, C, type, param_type, gate_kind) || !(eps >= 0.0f)) return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !residual || !h || !y || (gate_kind != LDN_GATE_NONE && !gate)) return kBadArgument;
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const SandwichArgs a = {x, residual, gate, pitch, pitch_residual, pitch_gate, rows, C,
                            {scale, post_weight, post_bias, weight, bias, param_type == LDN_F32}, eps, h, y, stats};
    if (with_type(type, [&](auto t) { return sandwich_rows<decltype(t)>(static_cast<Gate>(gate_kind), a, ctx, st, &r) ? 1 : 0; })) return r;
    const long long most = 32LL * ctx->sm_count;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return with_gate(static_cast<Gate>(gate_kind), [&](auto g) {
            return launch_after(sandwich_rows_kernel<T, decltype(g)::value>, static_cast<unsigned>(rows < most ? rows : most), kRowThreads, 0, st, a);
        });
    });
}

extern "C" LDN_API int ldn_sandwich_norm_backward(const void* grad_y, const void* grad_h, const void* x, long long pitch, const void* h,
                                                  const void* gate, long long pitch_gate, int gate_kind, long long rows, int C, int type,
                                                  const void* scale, const void* post_weight, const void* post_bias, const void* weight,
                                                  int param_type, const float* stats, void* grad_x, void* grad_residual, void* grad_gate,
                                                  void* grad_scale, void* grad_post_weight, void* grad_post_bias, void* grad_weight,
                                                  void* grad_bias, ldn_stream_t stream) {
    if (!sandwich_fits(rows, C, type, param_type, gate_kind)) return kBadArgument;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool wide = param_type == LDN_F32;
    FoldArgs f = {nullptr, 0, C, {scale, post_weight, post_bias, weight, nullptr, wide}, grad_scale, grad_post_weight, grad_post_bias,
                  grad_weight, grad_bias};
    int r = kOk;
    if (rows == 0) {
        for (void* p : {grad_scale, grad_post_weight, grad_post_bias, grad_weight, grad_bias})
            if (p && r == kOk) r = cuda_status(cudaMemsetAsync(p, 0, static_cast<size_t>(C) * (wide ? 4 : size_of(type)), st));
        return r;
    }
    if ((!grad_y && !grad_h) || !x || !h || !stats || (gate_kind != LDN_GATE_NONE && !gate)) return kBadArgument;
    const DeviceCtx* ctx;
    if ((r = get_device_ctx(&ctx)) != kOk) return r;
    const Gate kind = static_cast<Gate>(gate_kind);
    SandwichGradArgs a = {grad_y, grad_h, x, h, gate, pitch, pitch_gate, rows, C, f.p, stats, grad_x, grad_residual, grad_gate, nullptr, nullptr};
    const int columns = (C + kColumns - 1) / kColumns;
    const bool sums = grad_scale || grad_post_weight || grad_post_bias || grad_weight || grad_bias;
    auto in_registers = [&](int* blocks, const cudaStream_t* st) {
        return with_type(type, [&](auto t) {
            using T = decltype(t);
            return grad_y ? sandwich_grad_rows<T, true>(kind, a, ctx, blocks, st) : sandwich_grad_rows<T, false>(kind, a, ctx, blocks, st);
        });
    };
    const bool registers = in_registers(&f.count, nullptr) == kOk;
    if (!registers) {
        const long long most = (4LL * ctx->sm_count + columns - 1) / columns, needed = (rows + 63) / 64;
        f.count = static_cast<int>(most < needed ? most : needed);
    }
    const size_t row_bytes = registers ? 0 : pad256(static_cast<size_t>(rows) * 2 * sizeof(float));
    const size_t part_bytes = sums ? static_cast<size_t>(f.count) * 4 * C * sizeof(float) : 0;
    Scratch scratch;
    if (row_bytes + part_bytes) {
        if ((r = scratch.take(st, row_bytes + part_bytes)) != kOk) return r;
        a.row_sums = reinterpret_cast<float*>(scratch.base);
        if (sums) f.parts = a.parts = reinterpret_cast<float*>(scratch.base + row_bytes);
    }
    if (registers && (r = in_registers(nullptr, &st)) != kOk) return r;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        int s = kOk;
        if (!registers)
            s = with_gate(kind, [&](auto g) {
                constexpr Gate G = decltype(g)::value;
                const long long most = 32LL * ctx->sm_count;
                const int q = launch_after(sandwich_grad_rows_kernel<T, G>, static_cast<unsigned>(rows < most ? rows : most), kRowThreads, 0, st, a);
                if (q != kOk || !sums) return q;
                return launch_after(sandwich_grad_columns_kernel<T, G>, dim3(columns, static_cast<unsigned>(f.count)), kColumns * kColumnLanes, 0,
                                    st, a);
            });
        if (s != kOk || !sums) return s;
        return launch_after(sandwich_fold_kernel<T>, columns, kColumns * 4 * kFoldLanes, 0, st, f);
    });
}
