// Layer norm of rows, alone and behind a dropout onto a residual stream:
//     h = residual + dropout(x) (or x),   y = (h - mean) / sqrt(mean((h - mean)^2) + eps) * weight + bias,
// its gradients, and the form that leaves a row as 8-bit integers with a scale for the integer product (ldn_int8.cu).
//
// Statistics are those of two passes (the mean first, then the squares of what is left), in 32 bits: rows with a large mean lose
// nothing.  h is held in the type of the activations, and what is held is what is normalised, so the backward pass sees the
// numbers that the forward pass used.
#include "ldn_norm.cuh"

namespace ldn {
namespace {

constexpr int kRowThreads = 256;

// Any length, alignment and pitch: a block per row, one element per thread and step; the row is read again for every pass
// (16384 x 5120 bf16 with a pitch of 5121: 166 us; 3355 x 20000: 250).
template <class T, Form F>
__global__ void __launch_bounds__(kRowThreads) norm_rows_kernel(NormArgs a) {
    stream_order_wait();  // (quantised rows: what comes behind may read what was there before this kernel)
    stream_order_release();
    __shared__ float slots[kRowThreads / 32];
    Generator gen;
    if constexpr (F == Form::Joined) gen = generator_of(a.drop);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.pitch;
        const long long at = row * a.C;
        float sum = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            float v = to_float(x[c]);
            if constexpr (F == Form::Joined) {
                v = __fadd_rn(to_float(static_cast<const T*>(a.residual)[row * a.pitch_residual + c]),
                              dropped(a.drop, random_word(gen, at + c), v));
                static_cast<T*>(a.h)[at + c] = from_float<T>(v);
                v = rounded<T>(v);
            }
            sum += v;
        }
        if constexpr (F == Form::Joined) x = static_cast<const T*>(a.h) + at;  // (a thread reads back what it wrote)
        float mean = 0.0f, rstd = 0.0f;
        if constexpr (F != Form::Quantised) {
            mean = block_sum(sum, slots) / a.C;
            float squares = 0.0f;
            for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
                const float d = to_float(x[c]) - mean;
                squares += d * d;
            }
            rstd = 1.0f / sqrtf(block_sum(squares, slots) / a.C + a.eps);
        }
        if (threadIdx.x == 0 && a.mean) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        auto normed = [&](int c) {
            if (F == Form::Quantised) return to_float(x[c]);
            float v = (to_float(x[c]) - mean) * rstd;
            if (a.weight) v *= param_at<T>(a.weight, a.wide, c);
            return a.bias ? v + param_at<T>(a.bias, a.wide, c) : v;
        };
        if constexpr (F == Form::Integers || F == Form::Quantised) {
            unsigned largest = 0;
            for (int c = threadIdx.x; c < a.C; c += kRowThreads) largest = max(largest, magnitude(normed(c)));
            __shared__ unsigned all;
            __syncthreads();
            if (threadIdx.x == 0) all = 0;
            __syncthreads();
            atomicMax(&all, largest);
            __syncthreads();
            const float step = step_of(all), inverse = 1.0f / step;
            for (int c = threadIdx.x; c < a.C; c += kRowThreads)
                a.q[row * a.pitch_q + c] = static_cast<signed char>(steps(normed(c), inverse));
            if (threadIdx.x == 0) a.scale[row] = step;
        } else {
            for (int c = threadIdx.x; c < a.C; c += kRowThreads) static_cast<T*>(a.y)[at + c] = from_float<T>(normed(c));
        }
    }
}

// a = grad_y * weight, z = (x - mean) rstd:  grad_x = rstd (a - mean(a) - z mean(a z))
// (16384 x 5120 bf16 with a pitch of 5121, with the columns' sums: 394 us; 3355 x 20000: 390)
template <class T, bool JOINED>
__global__ void __launch_bounds__(kRowThreads) norm_grad_rows_kernel(NormGradArgs a) {
    stream_order_begin();
    __shared__ float slots[kRowThreads / 32];
    Generator gen;
    if constexpr (JOINED) gen = generator_of(a.drop);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.pitch;
        const long long at = row * a.C;
        const T* gy = static_cast<const T*>(a.grad_y) + at;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s = 0.0f, sz = 0.0f;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            const float g = to_float(gy[c]) * (a.weight ? param_at<T>(a.weight, a.wide, c) : 1.0f);
            s += g;
            sz += g * ((to_float(x[c]) - mean) * rstd);
        }
        s = block_sum(s, slots) / a.C;
        sz = block_sum(sz, slots) / a.C;
        for (int c = threadIdx.x; c < a.C; c += kRowThreads) {
            const float g = to_float(gy[c]) * (a.weight ? param_at<T>(a.weight, a.wide, c) : 1.0f);
            float v = rstd * (g - s - (to_float(x[c]) - mean) * rstd * sz);
            if constexpr (JOINED) {
                if (a.grad_h) v += to_float(static_cast<const T*>(a.grad_h)[at + c]);
                if (a.grad_residual) static_cast<T*>(a.grad_residual)[at + c] = from_float<T>(v);
                v = dropped(a.drop, random_word(gen, at + c), v);
            }
            if (a.grad_x) static_cast<T*>(a.grad_x)[at + c] = from_float<T>(v);
        }
    }
}

constexpr int kColumns = 32, kColumnLanes = 8;

// Column sums of grad_y z and grad_y over a block of rows: a thread has a column and every eighth row.
template <class T>
__global__ void __launch_bounds__(kColumns * kColumnLanes) norm_grad_columns_kernel(NormGradArgs a) {
    stream_order_begin();
    __shared__ float sums[2][kColumnLanes][kColumns];
    const int lane = threadIdx.x % kColumns, part = threadIdx.x / kColumns, c = blockIdx.x * kColumns + lane;
    const long long first = a.rows * blockIdx.y / gridDim.y, last = a.rows * (blockIdx.y + 1) / gridDim.y;
    float w = 0.0f, b = 0.0f;
    if (c < a.C)
        for (long long row = first + part; row < last; row += kColumnLanes) {
            const float g = to_float(static_cast<const T*>(a.grad_y)[row * a.C + c]);
            w += g * ((to_float(static_cast<const T*>(a.x)[row * a.pitch + c]) - a.mean[row]) * a.rstd[row]);
            b += g;
        }
    sums[0][part][lane] = w;
    sums[1][part][lane] = b;
    __syncthreads();
    if (part < 2 && c < a.C) {
        float s = 0.0f;
        for (int i = 0; i < kColumnLanes; ++i) s += sums[part][i][lane];
        a.parts[(static_cast<long long>(blockIdx.y) * 2 + part) * a.C + c] = s;
    }
}

// The parts in order: a thread has a column of one of the two sums and every 16th part, ten of them under way.  Blocks are small
// enough for all of them to be on the device at once (of 1024 threads, the last ones of 5120 columns came in a second wave: 9 us).
constexpr int kFoldLanes = 16, kFoldAhead = 10;
template <class T>
__global__ void __launch_bounds__(kColumns * kFoldLanes) norm_grad_fold_kernel(const float* parts, int count, int C, bool wide,
                                                                               void* grad_weight, void* grad_bias) {
    stream_order_begin();
    __shared__ float sums[kFoldLanes][kColumns + 1];
    const int lane = threadIdx.x % kColumns, part = threadIdx.x / kColumns, c = blockIdx.x * kColumns + lane;
    const float* from = parts + static_cast<long long>(blockIdx.y) * C + c;
    float s = 0.0f;
    if (c < C)
        for (int i = part; i < count; i += kFoldAhead * kFoldLanes) {
            float v[kFoldAhead];
#pragma unroll
            for (int u = 0; u < kFoldAhead; ++u) {
                const int k = i + u * kFoldLanes;
                v[u] = k < count ? from[2LL * k * C] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < kFoldAhead; ++u) s += v[u];
        }
    sums[part][lane] = s;
    __syncthreads();
    // a warp adds up two columns' sums, half of it each
    const int column = 2 * part + lane / kFoldLanes;
    s = sums[lane % kFoldLanes][column];
#pragma unroll
    for (int d = kFoldLanes / 2; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    void* to = blockIdx.y == 0 ? grad_weight : grad_bias;
    if (lane % kFoldLanes == 0 && blockIdx.x * kColumns + column < C && to) set_param<T>(to, wide, blockIdx.x * kColumns + column, s);
}

bool params_fit(int type, int param_type, const void* weight, const void* bias) {
    return (!weight && !bias) || param_type == LDN_F32 || param_type == type;
}

}  // namespace

template <Form F>
int norm_forward(const NormArgs& a, int type, cudaStream_t st) {
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    if (norm_in_registers(F, a, type, ctx, st, &r)) return r;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const long long most = 32LL * ctx->sm_count;
        return launch_after(norm_rows_kernel<T, F>, static_cast<unsigned>(a.rows < most ? a.rows : most), kRowThreads, 0, st, a);
    });
}

template int norm_forward<Form::Quantised>(const NormArgs& a, int type, cudaStream_t st);

namespace {

int zero_param(void* p, bool wide, int type, int C, cudaStream_t st) {
    return p ? cuda_status(cudaMemsetAsync(p, 0, static_cast<size_t>(C) * (wide ? 4 : size_of(type)), st)) : kOk;
}

template <bool JOINED>
int norm_backward(NormGradArgs a, int type, void* grad_weight, void* grad_bias, cudaStream_t st) {
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    if (a.rows == 0) {
        r = zero_param(grad_weight, a.wide, type, a.C, st);
        return r == kOk ? zero_param(grad_bias, a.wide, type, a.C, st) : r;
    }
    const int columns = (a.C + kColumns - 1) / kColumns;
    const bool sums = grad_weight || grad_bias;
    int blocks = 0;
    const bool registers = norm_grad_in_registers(JOINED, a, type, ctx, &blocks);
    if (!registers) {
        const long long most = (4LL * ctx->sm_count + columns - 1) / columns, needed = (a.rows + 63) / 64;
        blocks = static_cast<int>(most < needed ? most : needed);
    }
    Scratch scratch;
    if (sums) {
        r = scratch.take(st, static_cast<size_t>(blocks) * 2 * a.C * sizeof(float));
        if (r != kOk) return r;
        a.parts = reinterpret_cast<float*>(scratch.base);
    }
    if (registers) r = launch_norm_grad_in_registers(JOINED, a, type, ctx, st);
    if (r != kOk) return r;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const long long most = 32LL * ctx->sm_count;
        int r = kOk;
        if (!registers && (a.grad_x || a.grad_residual))
            r = launch_after(norm_grad_rows_kernel<T, JOINED>, static_cast<unsigned>(a.rows < most ? a.rows : most), kRowThreads, 0,
                             st, a);
        if (!sums || r != kOk) return r;
        if (!registers)
            r = launch_after(norm_grad_columns_kernel<T>, dim3(columns, static_cast<unsigned>(blocks)), kColumns * kColumnLanes, 0, st, a);
        if (r != kOk) return r;
        return launch_after(norm_grad_fold_kernel<T>, dim3(columns, 2), kColumns * kFoldLanes, 0, st, a.parts, blocks, a.C, a.wide,
                            grad_weight, grad_bias);
    });
}

}  // namespace
}  // namespace ldn

using namespace ldn;

extern "C" LDN_API int ldn_layer_norm(const void* x, long long pitch, long long rows, int C, int type, const void* weight,
                                      const void* bias, int param_type, float eps, void* y, float* mean, float* rstd,
                                      ldn_stream_t stream) {
    if (rows < 0 || !row_fits(C) || !known_type(type) || !params_fit(type, param_type, weight, bias) || !(eps >= 0.0f) || !mean != !rstd)
        return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !y) return kBadArgument;
    NormArgs a = {};
    a.x = x; a.pitch = pitch; a.rows = rows; a.C = C;
    a.weight = weight; a.bias = bias; a.wide = param_type == LDN_F32; a.eps = eps;
    a.y = y; a.mean = mean; a.rstd = rstd;
    return norm_forward<Form::Plain>(a, type, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LDN_API int ldn_layer_norm_backward(const void* grad_y, const void* x, long long pitch, long long rows, int C, int type,
                                               const float* mean, const float* rstd, const void* weight, int param_type,
                                               void* grad_x, void* grad_weight, void* grad_bias, ldn_stream_t stream) {
    if (rows < 0 || !row_fits(C) || !known_type(type) || !known_type(param_type) || !params_fit(type, param_type, weight, grad_weight))
        return kBadArgument;
    if (rows > 0 && (!grad_y || !x || !mean || !rstd)) return kBadArgument;
    NormGradArgs a = {};
    a.grad_y = grad_y; a.x = x; a.pitch = pitch; a.rows = rows; a.C = C;
    a.mean = mean; a.rstd = rstd; a.weight = weight; a.wide = param_type == LDN_F32;
    a.grad_x = grad_x;
    return norm_backward<false>(a, type, grad_weight, grad_bias, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LDN_API int ldn_dropout_add_layer_norm(const void* x, long long pitch, const void* residual, long long pitch_residual,
                                                  long long rows, int C, int type, const void* weight, const void* bias,
                                                  int param_type, float eps, double p, unsigned long long seed,
                                                  unsigned long long offset, const unsigned long long* state, void* h, void* y,
                                                  float* mean, float* rstd, ldn_stream_t stream) {
    NormArgs a = {};
    if (rows < 0 || !row_fits(C) || !known_type(type) || !params_fit(type, param_type, weight, bias) || !(eps >= 0.0f) ||
        !mean != !rstd || !make_dropout(p, seed, offset, state, &a.drop))
        return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !residual || !h || !y) return kBadArgument;
    a.x = x; a.pitch = pitch; a.residual = residual; a.pitch_residual = pitch_residual; a.rows = rows; a.C = C;
    a.weight = weight; a.bias = bias; a.wide = param_type == LDN_F32; a.eps = eps;
    a.h = h; a.y = y; a.mean = mean; a.rstd = rstd;
    return norm_forward<Form::Joined>(a, type, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LDN_API int ldn_dropout_add_layer_norm_backward(const void* grad_y, const void* grad_h, const void* h, long long rows,
                                                           int C, int type, const float* mean, const float* rstd,
                                                           const void* weight, int param_type, double p, unsigned long long seed,
                                                           unsigned long long offset, const unsigned long long* state,
                                                           void* grad_x, void* grad_residual, void* grad_weight, void* grad_bias,
                                                           ldn_stream_t stream) {
    NormGradArgs a = {};
    if (rows < 0 || !row_fits(C) || !known_type(type) || !known_type(param_type) || !params_fit(type, param_type, weight, grad_weight) ||
        !make_dropout(p, seed, offset, state, &a.drop))
        return kBadArgument;
    if (rows > 0 && (!grad_y || !h || !mean || !rstd)) return kBadArgument;
    a.grad_y = grad_y; a.grad_h = grad_h; a.x = h; a.pitch = C; a.rows = rows; a.C = C;
    a.mean = mean; a.rstd = rstd; a.weight = weight; a.wide = param_type == LDN_F32;
    a.grad_x = grad_x; a.grad_residual = grad_residual;
    return norm_backward<true>(a, type, grad_weight, grad_bias, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LDN_API int ldn_layer_norm_quantized(const void* x, long long pitch, long long rows, int C, int type, const void* weight,
                                                const void* bias, int param_type, float eps, signed char* q, long long pitch_q,
                                                float* scale, ldn_stream_t stream) {
    if (rows < 0 || !row_fits(C) || !known_type(type) || !params_fit(type, param_type, weight, bias) || !(eps >= 0.0f) || pitch_q < C)
        return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !q || !scale) return kBadArgument;
    NormArgs a = {};
    a.x = x; a.pitch = pitch; a.rows = rows; a.C = C;
    a.weight = weight; a.bias = bias; a.wide = param_type == LDN_F32; a.eps = eps;
    a.q = q; a.pitch_q = pitch_q; a.scale = scale;
    return norm_forward<Form::Integers>(a, type, reinterpret_cast<cudaStream_t>(stream));
}
