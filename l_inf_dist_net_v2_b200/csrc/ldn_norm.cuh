// Layer norm as its kernels see it.
#pragma once
#include "ldn_head.cuh"

namespace ldn {

// What leaves a row kernel: the norm; the norm of residual + dropout; the norm as integers; the row itself as integers
enum class Form { Plain, Joined, Integers, Quantised };

struct NormArgs {
    const void* x;
    const void* residual;  // joined form only
    long long pitch, pitch_residual, rows;
    int C;
    const void *weight, *bias;  // may be null
    bool wide;                  // they have 32 bits
    float eps;
    DropoutArgs drop;
    void *h, *y;
    float *mean, *rstd;  // may be null
    signed char* q;      // integer forms only
    long long pitch_q;
    float* scale;
};

struct NormGradArgs {
    const void* grad_y;  // rows of C
    const void* grad_h;  // joined form only, may be null
    const void* x;       // what was normalised
    long long pitch, rows;
    int C;
    const float *mean, *rstd;
    const void* weight;
    bool wide;
    DropoutArgs drop;
    void* grad_x;         // may be null
    void* grad_residual;  // joined form only: the gradient of h; may be null
    float* parts;         // [block of rows][2][C]: sums for the weight and the bias; may be null
};

// All of it (ldn_norm.cu): arguments checked, at least one row
template <Form F>
int norm_forward(const NormArgs& a, int type, cudaStream_t st);

// Rows held in registers; false: these rows do not fit, or their tensors' pieces do not match
bool norm_in_registers(Form form, const NormArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st, int* status);
// The same for the gradient, whose sums over blocks of rows are `blocks` parts; plan first, then launch with room for them
bool norm_grad_in_registers(bool joined, const NormGradArgs& a, int type, const DeviceCtx* ctx, int* blocks);
int launch_norm_grad_in_registers(bool joined, const NormGradArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st);

}  // namespace ldn
