// Matrix product in 8-bit integers with a scale per token and per output channel:
//     out[m, n] = act(sum_k q[m, k] w[n, k] * scale[m] * w_scale[n] + bias[n]),
// the sums exact in 32-bit integers, the rest in 32-bit floating point; and rows as such integers.
#include "ldn_int8.cuh"
#include "ldn_norm.cuh"

namespace ldn {
namespace {

constexpr int kMostTerms = 131071;  // 2^31 / 2^14: sums of products of two values of -128 .. 127 stay in 32 bits

// Rows of bytes that start anywhere as rows that start at multiples of 16 bytes
__global__ void __launch_bounds__(kThreads) align_rows_kernel(const signed char* from, long long pitch, long long rows, int C,
                                                              signed char* to, long long pitch_to) {
    stream_order_begin();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x)
        for (int c = threadIdx.x; c < C; c += kThreads) to[row * pitch_to + c] = from[row * pitch + c];
}

int launch_quantize(const void* x, long long pitch, long long rows, int C, int type, signed char* q, long long pitch_q, float* scale,
                    cudaStream_t st) {
    NormArgs a = {};
    a.x = x; a.pitch = pitch; a.rows = rows; a.C = C;
    a.q = q; a.pitch_q = pitch_q; a.scale = scale;
    return norm_forward<Form::Quantised>(a, type, st);
}

long long padded16(long long bytes) { return (bytes + 15) / 16 * 16; }
bool aligned_rows(const void* p, long long pitch) { return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(pitch)) & 15u) == 0; }

// Scratch of a product: the operands that have to be copied, as the tiles' loads want them
struct Operands {
    bool copy_q, copy_w;
    size_t bytes_q, bytes_w;
};
Operands operands_of(const ProductArgs& a) {
    Operands o = {!aligned_rows(a.q, a.pitch_q), !aligned_rows(a.w, a.pitch_w), 0, 0};
    if (o.copy_q) o.bytes_q = pad256(static_cast<size_t>(a.M) * padded16(a.K));
    if (o.copy_w) o.bytes_w = pad256(static_cast<size_t>(a.N) * padded16(a.K));
    return o;
}
int launch_align(const signed char** p, long long* pitch, long long rows, int K, char* to, const DeviceCtx* ctx, cudaStream_t st) {
    const long long most = 32LL * ctx->sm_count;
    signed char* q = reinterpret_cast<signed char*>(to);
    const int r = launch_after(align_rows_kernel, static_cast<unsigned>(rows < most ? rows : most), kThreads, 0, st, *p, *pitch, rows, K,
                               q, padded16(K));
    *p = q;
    *pitch = padded16(K);
    return r;
}

int launch_product(ProductArgs a, int type, const Operands& o, char* scratch, int* status, const DeviceCtx* ctx, cudaStream_t st) {
    int r = kOk;
    if (o.copy_q) r = launch_align(&a.q, &a.pitch_q, a.M, a.K, scratch, ctx, st);
    if (r == kOk && o.copy_w) r = launch_align(&a.w, &a.pitch_w, a.N, a.K, scratch + o.bytes_q, ctx, st);
    return r == kOk ? launch_product_tiles(a, type, status, ctx, st) : r;
}

bool product_fits(long long M, int N, int K, int activation, int type, long long pitch_w) {
    return M >= 0 && row_fits(N) && K > 0 && K <= kMostTerms && activation >= LDN_NO_ACTIVATION && activation <= LDN_TANH &&
           known_type(type) && pitch_w >= K;
}

}  // namespace
}  // namespace ldn

using namespace ldn;

extern "C" LDN_API int ldn_quantize_rows(const void* x, long long pitch, long long rows, int C, int type, signed char* q,
                                         long long pitch_q, float* scale, ldn_stream_t stream) {
    if (rows < 0 || !row_fits(C) || !known_type(type) || pitch_q < C) return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !q || !scale) return kBadArgument;
    return launch_quantize(x, pitch, rows, C, type, q, pitch_q, scale, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LDN_API int ldn_int8_linear(const signed char* q, long long pitch_q, const float* scale, const signed char* w,
                                       long long pitch_w, const float* w_scale, const float* bias, long long M, int N, int K,
                                       int activation, void* out, int type, ldn_stream_t stream) {
    if (!product_fits(M, N, K, activation, type, pitch_w) || pitch_q < K) return kBadArgument;
    if (M == 0) return kOk;
    if (!q || !scale || !w || !w_scale || !out) return kBadArgument;
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const ProductArgs a = {q, pitch_q, scale, w, pitch_w, w_scale, bias, M, N, K, activation, out};
    if (product_is_single(a)) return launch_product_single(a, nullptr, 0, type, type, ctx, st);
    const Operands o = operands_of(a);
    Scratch scratch;
    if ((r = scratch.take(st, o.bytes_q + o.bytes_w)) != kOk) return r;
    return launch_product(a, type, o, scratch.base, scratch.status, ctx, st);
}

extern "C" LDN_API int ldn_int8_linear_float(const void* x, long long pitch, int x_type, const signed char* w, long long pitch_w,
                                             const float* w_scale, const float* bias, long long M, int N, int K, int activation,
                                             void* out, int type, ldn_stream_t stream) {
    if (!product_fits(M, N, K, activation, type, pitch_w) || !known_type(x_type)) return kBadArgument;
    if (M == 0) return kOk;
    if (!x || !w || !w_scale || !out) return kBadArgument;
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const long long pitch_q = padded16(K);
    const size_t bytes_q = pad256(static_cast<size_t>(M) * pitch_q), bytes_scale = pad256(sizeof(float) * static_cast<size_t>(M));
    ProductArgs a = {nullptr, pitch_q, nullptr, w, pitch_w, w_scale, bias, M, N, K, activation, out};
    if (product_is_single(a)) return launch_product_single(a, x, pitch, x_type, type, ctx, st);
    const Operands o = operands_of(a);
    Scratch scratch;
    if ((r = scratch.take(st, bytes_q + bytes_scale + o.bytes_w)) != kOk) return r;
    signed char* q = reinterpret_cast<signed char*>(scratch.base);
    float* scale = reinterpret_cast<float*>(scratch.base + bytes_q);
    if ((r = launch_quantize(x, pitch, M, K, x_type, q, pitch_q, scale, st)) != kOk) return r;
    a.q = q;
    a.scale = scale;
    a.w_early = !o.copy_w;
    return launch_product(a, type, o, scratch.base + bytes_q + bytes_scale, scratch.status, ctx, st);
}
