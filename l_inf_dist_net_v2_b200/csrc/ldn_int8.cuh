// The integer product as its kernels see it.
#pragma once
#include "ldn_head.cuh"

namespace ldn {

struct ProductArgs {
    const signed char* q;  // [M][pitch_q]
    long long pitch_q;
    const float* scale;
    const signed char* w;  // [N][pitch_w]
    long long pitch_w;
    const float *w_scale, *bias;
    long long M;
    int N, K, activation;
    void* out;  // [M][N]
    bool w_early = false;  // the weight may be read before the kernel in front is done: that is this call's own quantising, which lets
                           // this one begin only when all in front of it is
};

#ifdef __CUDACC__
// (called, not inlined: sixteen copies of it in a loop over a thread's sums came from memory every time and cost more than the
// products)
static __device__ __noinline__ float tanh_called(float v) { return tanhf(v); }
__device__ __forceinline__ float product_value(int sum, float scale, float w_scale, float bias, int activation) {
    const float v = fmaf(__fmul_rn(static_cast<float>(sum), scale), w_scale, bias);
    return activation == LDN_RELU ? (v < 0.0f ? 0.0f : v) : activation == LDN_TANH ? tanh_called(v) : v;
}
// What follows the sums of one output for N tokens, two at a time and without a branch per value (values in flight hide each
// other's latency); bias: 0 where there is none
template <int N>
__device__ __forceinline__ void product_values(const int (&sum)[N], const float (&scale)[N], float w_scale, float bias, int activation,
                                               float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const float2 s = make_float2(static_cast<float>(sum[j]), static_cast<float>(sum[j + 1]));
        const float2 r = __ffma2_rn(__fmul2_rn(s, make_float2(scale[j], scale[j + 1])), make_float2(w_scale, w_scale), make_float2(bias, bias));
        v[j] = r.x;
        v[j + 1] = r.y;
    }
    if (activation == LDN_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];  // (what is not a number stays)
    } else if (activation == LDN_TANH) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = tanh_called(v[j]);
    }
}
#endif

// Both operands' rows start at multiples of 16 bytes
int launch_product_tiles(const ProductArgs& a, int type, int* status, const DeviceCtx* ctx, cudaStream_t st);

// One to four tokens, the weight's rows at multiples of 16 bytes; x: rows of x_type to be quantised, or null (the product's integers)
bool product_is_single(const ProductArgs& a);
int launch_product_single(const ProductArgs& a, const void* x, long long pitch, int x_type, int out_type, const DeviceCtx* ctx,
                          cudaStream_t st);

}  // namespace ldn
