// The gated projection of a head's block as its kernels see it:
//     y = act(g) u,   g = x Wg' + bg,   u = x Wu' + bu,
// and with the incoming gradient dy: dg = dy u act'(g), du = dy act(g), dx = dg Wg + du Wu, dWg = dg' x, dWu = du' x, the biases'
// gradients the column sums of dg and du.
#pragma once
#include "ldn_head.cuh"

namespace ldn {

struct GatedArgs {
    const void* x;  // [T][pitch_x]
    long long pitch_x;
    const void *w_gate, *w_up;  // [H][pitch]
    long long pitch_gate, pitch_up;
    const void *b_gate, *b_up;  // may be null
    bool wide;                  // they have 32 bits
    long long T;
    int K, H, activation;
    void* y;              // [T][H]
    float *g, *u;           // [T][pitch_saved], kept for the backward pass; may be null
    long long pitch_saved;  // a multiple of 16, as the addresses are of 32 bytes
};

inline bool gated_activation(int a) { return a == LDN_RELU || a == LDN_SILU || a == LDN_GELU || a == LDN_SIGMOID; }

// A handful of rows, without tensor cores (ldn_gated_rows.cu)
bool gated_is_few(const GatedArgs& a, int type);
int launch_gated_few(const GatedArgs& a, int type, cudaStream_t st);

// ---- products on the tensor cores (ldn_gated_tiles.cu) --------------------------------------------------------------------------
// An operand as the tensor cores' loads want it: [image][row][pitch] of 16 bits, rows at multiples of 16 bytes.  32-bit operands are three
// bfloat16 images each, whose sum they are.
struct Images {
    const void* base = nullptr;
    long long rows = 0;
    int columns = 0;
    long long pitch = 0;  // elements
    int count = 1;
    long long apart = 0;  // elements between images
};
enum class GatedForm {
    Forward,     // [T][H] from rows x K, both projections side by side
    GradRows,    // [T][K] from dg, du (images of one operand) and the projections
    GradWeights  // 2 x [H][K] from dg, du and x
};
struct TileArgs {
    long long M;  // rows of an output
    int N;        // its columns
    int tiles_m, tiles_n;
    int tiles, whole, pairs;  // of the tiles, how many a pair of CTAs takes as a whole; the rest are shared out in units
    int units, side_units, side_steps;
    bool drained;  // sums of 16-bit products leave the accumulator after every unit
    const void *b_gate, *b_up;
    bool wide;
    int activation;
    void *out0, *out1, *out2;
    long long pitch, pitch_saved;  // of out0 (GradWeights: of both), of what is kept
    float* partials;
    int* status;
};
// Scratch for the parts of tiles that several pairs share; `a`, `b0`, `b1`: the operands, b1 for the up projection
size_t gated_tiles_scratch(GatedForm form, long long M, int N, int terms, int type, const DeviceCtx* ctx);
int launch_gated_tiles(GatedForm form, TileArgs a, int terms, const Images& op_a, const Images& op_b0, const Images& op_b1, int type,
                       char* scratch, int* status, const DeviceCtx* ctx, cudaStream_t st);

#ifdef __CUDACC__
// 1 / (1 + e^-g); the quotient's error is 2 units at most, and it is 0 where e^-g has no number
__device__ __forceinline__ float logistic(float g) { return __fdividef(1.0f, 1.0f + expf(-g)); }
// The normal distribution's function, and e^(-g^2 / 2).  With t = |g|, the smaller of the function's two sides is e^(-t^2 / 2) q(t), q falling
// from 1/2 to 0.4 / t: u P(u) with u = 1 / (1 + 0.24 t), P of degree 9 fitted to q(t) / u over u(0 .. 20) for the least relative error, 4e-9.
// What t^2 is rounded by is put back.  A dozen units of 2^-24 of itself at most, on either side (0.5 (1 + erf) leaves nothing of it
// below -5.5).
struct Normal {
    float cdf, bell;
};
__device__ __forceinline__ Normal normal_of(float g) {
    float t;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"(fabsf(g)), "f"(20.0f));  // (both are 0 there)
    const float u = __fdividef(1.0f, fmaf(0.24f, t, 1.0f));
    float p = 0.025488367f;
    p = fmaf(p, u, -0.12448445f);
    p = fmaf(p, u, 0.20524898f);
    p = fmaf(p, u, -0.14414364f);
    p = fmaf(p, u, 0.14150542f);
    p = fmaf(p, u, 0.028033895f);
    p = fmaf(p, u, 0.0878384f);
    p = fmaf(p, u, 0.08890992f);
    p = fmaf(p, u, 0.0958613f);
    p = fmaf(p, u, 0.0957418f);
    const float square = __fmul_rn(t, t), rest = fmaf(t, t, -square);
    float bell = expf(-0.5f * square);
    bell = fmaf(bell, -0.5f * rest, bell);
    const float low = bell * (u * p);
    return {g < 0.0f ? low : 1.0f - low, bell};
}
// (called: see tanh_called of the integer product)
static __device__ __noinline__ float normal_cdf(float g) { return normal_of(g).cdf; }

// act(g) of N numbers
template <int N>
__device__ __forceinline__ void activate(float (&g)[N], int activation) {
    if (activation == LDN_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] *= logistic(g[j]);
    } else if (activation == LDN_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] *= normal_cdf(g[j]);
    } else if (activation == LDN_SIGMOID) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] = logistic(g[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] = g[j] < 0.0f ? 0.0f : g[j];  // (what is not a number stays)
    }
}
// act(g) and act'(g)
__device__ __forceinline__ float2 activation_and_slope(float g, int activation) {
    if (activation == LDN_RELU) return make_float2(g < 0.0f ? 0.0f : g, g > 0.0f ? 1.0f : 0.0f);
    if (activation == LDN_GELU) {
        const Normal n = normal_of(g);
        return make_float2(g * n.cdf, n.cdf + g * (0.39894228040143268f * n.bell));
    }
    // (s and 1 - s from e^-|g|, so that the smaller one keeps its digits)
    const float e = expf(-fabsf(g)), larger_one = __fdividef(1.0f, 1.0f + e), smaller_one = e * larger_one;
    const float s = g < 0.0f ? smaller_one : larger_one, rest = g < 0.0f ? larger_one : smaller_one;
    return activation == LDN_SIGMOID ? make_float2(s, s * rest) : make_float2(g * s, s * (1.0f + g * rest));
}
#endif

}  // namespace ldn
