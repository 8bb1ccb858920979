// Matrix product in 8-bit integers with a scale per token and per output channel:
//     out[m, n] = act(sum_k q[m, k] w[n, k] * scale[m] * w_scale[n] + bias[n]),
// the sums exact in 32-bit integers, the rest in 32-bit floating point; and rows as such integers.
#include "ldn_head.cuh"

namespace ldn {
namespace {

constexpr int kMostTerms = 131071;  // 2^31 / 2^14: sums of products of two values of -128 .. 127 stay in 32 bits

// A block per row: the largest magnitude, then the integers.
template <class T>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const void* x, long long pitch, long long rows, int C, signed char* q,
                                                                 long long pitch_q, float* scale) {
    stream_order_begin();
    __shared__ unsigned all;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* v = static_cast<const T*>(x) + row * pitch;
        unsigned largest = 0;
        for (int c = threadIdx.x; c < C; c += kThreads) largest = max(largest, magnitude(to_float(v[c])));
        __syncthreads();
        if (threadIdx.x == 0) all = 0;
        __syncthreads();
        atomicMax(&all, largest);
        __syncthreads();
        const float step = step_of(all), inverse = __frcp_rn(step);
        for (int c = threadIdx.x; c < C; c += kThreads) q[row * pitch_q + c] = static_cast<signed char>(steps(to_float(v[c]), inverse));
        if (threadIdx.x == 0) scale[row] = step;
    }
}

struct ProductArgs {
    const signed char* q;
    long long pitch_q;
    const float* scale;
    const signed char* w;
    long long pitch_w;
    const float *w_scale, *bias;
    long long M;
    int N, K, activation;
    void* out;
};

__device__ __forceinline__ float activated(float v, int activation) {
    if (activation == LDN_RELU) return v < 0.0f ? 0.0f : v;  // (what is not a number stays)
    return activation == LDN_TANH ? tanhf(v) : v;
}
__device__ __forceinline__ float product_value(const ProductArgs& a, int sum, float scale, int n) {
    float v = __fmul_rn(__fmul_rn(static_cast<float>(sum), scale), a.w_scale[n]);
    if (a.bias) v = __fadd_rn(v, a.bias[n]);
    return activated(v, a.activation);
}

// 64 x 64 outputs per block, 4 x 4 per thread, four products per instruction; any alignment.
constexpr int kSide = 64, kWords = 16;
template <class T>
__global__ void __launch_bounds__(kThreads) product_tiles_kernel(ProductArgs a) {
    stream_order_begin();
    __shared__ int tile_q[kSide][kWords + 1], tile_w[kSide][kWords + 1];
    const long long m0 = static_cast<long long>(blockIdx.y) * kSide;
    const int n0 = blockIdx.x * kSide, tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    int sum[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 4 * kWords) {
        for (int i = threadIdx.x; i < kSide * kWords; i += kThreads) {
            const int r = i / kWords, k = k0 + 4 * (i % kWords);
            unsigned vq = 0, vw = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (k + e < a.K && m0 + r < a.M) vq |= static_cast<unsigned>(static_cast<unsigned char>(a.q[(m0 + r) * a.pitch_q + k + e])) << 8 * e;
                if (k + e < a.K && n0 + r < a.N) vw |= static_cast<unsigned>(static_cast<unsigned char>(a.w[(n0 + r) * a.pitch_w + k + e])) << 8 * e;
            }
            tile_q[r][i % kWords] = static_cast<int>(vq);
            tile_w[r][i % kWords] = static_cast<int>(vw);
        }
        __syncthreads();
#pragma unroll 4
        for (int k = 0; k < kWords; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[i][j] = __dp4a(tile_q[tm + 16 * i][k], tile_w[tn + 16 * j][k], sum[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long m = m0 + tm + 16 * i;
        if (m >= a.M) continue;
        const float scale = a.scale[m];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tn + 16 * j;
            if (n < a.N) static_cast<T*>(a.out)[m * a.N + n] = from_float<T>(product_value(a, sum[i][j], scale, n));
        }
    }
}

int launch_quantize(const void* x, long long pitch, long long rows, int C, int type, signed char* q, long long pitch_q, float* scale,
                    const DeviceCtx* ctx, cudaStream_t st) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const long long most = 32LL * ctx->sm_count;
        return launch_after(quantize_rows_kernel<T>, static_cast<unsigned>(rows < most ? rows : most), kThreads, 0, st, x, pitch, rows,
                            C, q, pitch_q, scale);
    });
}

int launch_product(const ProductArgs& a, int type, cudaStream_t st) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        for (ProductArgs b = a; b.M > 0;) {  // (a grid's second dimension has 16 bits)
            const long long rows = b.M < kSide * 65535LL ? b.M : kSide * 65535LL;
            ProductArgs c = b;
            c.M = rows;
            const int r = launch_after(product_tiles_kernel<T>, dim3((c.N + kSide - 1) / kSide, static_cast<unsigned>((rows + kSide - 1) / kSide)),
                                       kThreads, 0, st, c);
            if (r != kOk) return r;
            b.M -= rows;
            b.q += rows * b.pitch_q;
            b.scale += rows;
            b.out = static_cast<T*>(b.out) + rows * b.N;
        }
        return static_cast<int>(kOk);
    });
}

bool product_fits(long long M, int N, int K, int activation, int type, long long pitch_w) {
    return M >= 0 && N > 0 && K > 0 && K <= kMostTerms && activation >= LDN_NO_ACTIVATION && activation <= LDN_TANH &&
           known_type(type) && pitch_w >= K;
}

}  // namespace
}  // namespace ldn

using namespace ldn;

extern "C" LDN_API int ldn_quantize_rows(const void* x, long long pitch, long long rows, int C, int type, signed char* q,
                                         long long pitch_q, float* scale, ldn_stream_t stream) {
    if (rows < 0 || C <= 0 || !known_type(type) || pitch_q < C) return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !q || !scale) return kBadArgument;
    const DeviceCtx* ctx;
    const int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    return launch_quantize(x, pitch, rows, C, type, q, pitch_q, scale, ctx, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" LDN_API int ldn_int8_linear(const signed char* q, long long pitch_q, const float* scale, const signed char* w,
                                       long long pitch_w, const float* w_scale, const float* bias, long long M, int N, int K,
                                       int activation, void* out, int type, ldn_stream_t stream) {
    if (!product_fits(M, N, K, activation, type, pitch_w) || pitch_q < K) return kBadArgument;
    if (M == 0) return kOk;
    if (!q || !scale || !w || !w_scale || !out) return kBadArgument;
    ProductArgs a = {q, pitch_q, scale, w, pitch_w, w_scale, bias, M, N, K, activation, out};
    return launch_product(a, type, reinterpret_cast<cudaStream_t>(stream));
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
    const long long pitch_q = (K + 15LL) / 16 * 16;
    const size_t bytes_q = pad256(static_cast<size_t>(M) * pitch_q);
    Scratch scratch;
    if ((r = scratch.take(st, bytes_q + sizeof(float) * static_cast<size_t>(M))) != kOk) return r;
    signed char* q = reinterpret_cast<signed char*>(scratch.base);
    float* scale = reinterpret_cast<float*>(scratch.base + bytes_q);
    if ((r = launch_quantize(x, pitch, M, K, x_type, q, pitch_q, scale, ctx, st)) != kOk) return r;
    ProductArgs a = {q, pitch_q, scale, w, pitch_w, w_scale, bias, M, N, K, activation, out};
    return launch_product(a, type, st);
}
