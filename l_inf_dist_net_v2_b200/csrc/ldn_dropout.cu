// Dropout with a counter-based generator: out = [residual +] (x / (1 - p) where its word says so, else 0).  No mask is stored;
// the backward pass is the same kernel on the gradient with the same seed and offset.
#include "ldn_head.cuh"

namespace ldn {
namespace {

struct DropoutCall {
    const void *x, *residual;
    long long pitch, pitch_residual, rows;
    int C;
    DropoutArgs drop;
    void* out;
};

// A thread has the four elements of a block of words, wherever the rows break.
template <class T>
__global__ void __launch_bounds__(kThreads) dropout_kernel(DropoutCall a) {
    stream_order_begin();
    const Generator gen = generator_of(a.drop);
    const long long n = a.rows * a.C, step = static_cast<long long>(gridDim.x) * kThreads;
    for (long long block = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; block * 4 < n; block += step) {
        const uint4 words = random_words(gen, block);
        const unsigned word[4] = {words.x, words.y, words.z, words.w};
        long long row = block * 4 / a.C;
        int c = static_cast<int>(block * 4 - row * a.C);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const long long i = block * 4 + e;
            if (i < n) {
                float v = dropped(a.drop, word[e], to_float(static_cast<const T*>(a.x)[row * a.pitch + c]));
                if (a.residual) v = __fadd_rn(to_float(static_cast<const T*>(a.residual)[row * a.pitch_residual + c]), v);
                static_cast<T*>(a.out)[i] = from_float<T>(v);
            }
            if (++c == a.C) {
                c = 0;
                ++row;
            }
        }
    }
}

}  // namespace
}  // namespace ldn

using namespace ldn;

extern "C" LDN_API int ldn_dropout(const void* x, long long pitch, const void* residual, long long pitch_residual, long long rows,
                                   int C, int type, double p, unsigned long long seed, unsigned long long offset,
                                   const unsigned long long* state, void* out, ldn_stream_t stream) {
    DropoutCall a = {};
    if (rows < 0 || C <= 0 || !known_type(type) || !make_dropout(p, seed, offset, state, &a.drop)) return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !out) return kBadArgument;
    const DeviceCtx* ctx;
    const int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    a.x = x; a.pitch = pitch; a.residual = residual; a.pitch_residual = pitch_residual; a.rows = rows; a.C = C; a.out = out;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const long long blocks = ((rows * C + 3) / 4 + kThreads - 1) / kThreads, most = 32LL * ctx->sm_count;
        return launch_after(dropout_kernel<T>, static_cast<unsigned>(blocks < most ? blocks : most), kThreads, 0,
                            reinterpret_cast<cudaStream_t>(stream), a);
    });
}
