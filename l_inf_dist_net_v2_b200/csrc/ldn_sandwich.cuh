// A block's result joined to the residual stream between two norms, as the kernels see it:
//     n = norm(x) post_weight + post_bias,   h = residual + gate scale n (held in the rows' type),   y = norm(h) weight + bias,
// norm(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps).  Backward, with z1, z2 the normalised rows and N(a, z) = a - mean(a) - z mean(a z):
//     d = dh + rstd2 N(dy weight, z2)   (the residual's gradient),   dgate = d scale n,   dx = rstd1 N(d gate scale post_weight, z1),
// and with the column sums P = sum d gate z1 and Q = sum d gate:
//     dpost_weight = scale P,   dpost_bias = scale Q,   dscale = post_weight P + post_bias Q;
// dweight = sum dy z2, dbias = sum dy.
#pragma once
#include "ldn_head.cuh"

namespace ldn {

enum class Gate { None = LDN_GATE_NONE, Row = LDN_GATE_ROW, All = LDN_GATE_ALL };

struct SandwichParams {
    const void *scale, *post_weight, *post_bias, *weight, *bias;  // may be null
    bool wide;                                                    // they have 32 bits
};
struct SandwichArgs {
    const void *x, *residual, *gate;
    long long pitch, pitch_residual, pitch_gate, rows;  // (a gate of one number per row has no pitch)
    int C;
    SandwichParams p;
    float eps;
    void *h, *y;
    float* stats;  // [4][rows]: mean and 1 / deviation of x, then of h; may be null
};
struct SandwichGradArgs {
    const void *grad_y, *grad_h;  // rows of C; either may be null (not both)
    const void *x, *h, *gate;
    long long pitch, pitch_gate, rows;  // of x; h has rows of C
    int C;
    SandwichParams p;
    const float* stats;
    void *grad_x, *grad_residual, *grad_gate;  // any may be null
    float* row_sums;  // [2][rows]: mean(a), mean(a z2); simple kernels
    float* parts;     // [block of rows][4][C]: sums of dy z2, dy, d gate z1, d gate; may be null
};

// Rows of T held in registers (ldn_sandwich_forward.cuh, ldn_sandwich_grad.cuh).  False: these rows do not fit, or their tensors' pieces do not match
template <class T>
bool sandwich_rows(Gate gate, const SandwichArgs& a, const DeviceCtx* ctx, cudaStream_t st, int* status);
// kOk: they do; blocks: how many parts of column sums they make, where not null; st: their launch, where not null.  OF_Y: grad_y is not null
template <class T, bool OF_Y>
int sandwich_grad_rows(Gate gate, const SandwichGradArgs& a, const DeviceCtx* ctx, int* blocks, const cudaStream_t* st);

#ifdef __CUDACC__
template <class T>
__device__ __forceinline__ float param_or(const void* p, bool wide, int c, float none) {
    return p ? param_at<T>(p, wide, c) : none;
}
#endif

}  // namespace ldn
