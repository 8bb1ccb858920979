// What the kernels of a head share (layer norm, dropout, the product in 8-bit integers): element types, the counter-based
// generator, sums over a block, and scratch from the stream's arena.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

#include "ldn_b200.h"
#include "ldn_common.cuh"

namespace ldn {

inline bool known_type(int type) { return type == LDN_F32 || type == LDN_F16 || type == LDN_BF16; }
inline int size_of(int type) { return type == LDN_F32 ? 4 : 2; }

// Calls f(T()) with the element type that `type` names; `type` is known.
template <class F>
int with_type(int type, F f) {
    switch (type) {
        case LDN_F32: return f(float());
        case LDN_F16: return f(__half());
        default: return f(__nv_bfloat16());
    }
}

// Scratch of one call, from the stream's arena; its lock is held for as long as the call enqueues work.
struct Scratch {
    std::unique_lock<std::mutex> lock;
    char* base = nullptr;
    int* status = nullptr;

    int take(cudaStream_t st, size_t bytes) {
        Arena* arena;
        int r = find_arena(st, &arena);
        if (r != kOk) return r;
        lock = std::unique_lock<std::mutex>(*static_cast<std::mutex*>(arena->call_mutex));
        if ((r = ensure_arena(arena, st, bytes)) != kOk) return r;
        arena->extreme_words = arena->power_words[0] = arena->power_words[1] = nullptr;  // (they lie in what this call overwrites)
        base = arena->base;
        status = arena->status;
        return kOk;
    }
};

// Dropout as a kernel sees it: element i of the logical array is kept if its word is at least `threshold`, and multiplied by
// `scale` then.  state (may be null): a seed and an offset on the device, in place of `seed` and in front of `offset`.
struct DropoutArgs {
    unsigned long long seed, offset;
    const unsigned long long* state;
    unsigned threshold;
    float scale;
    bool all;  // p = 1: nothing is kept
};
inline bool make_dropout(double p, unsigned long long seed, unsigned long long offset, const unsigned long long* state, DropoutArgs* d) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    const double words = p * 4294967296.0;
    d->seed = seed;
    d->offset = offset;
    d->state = state;
    d->all = words >= 4294967295.5;
    d->threshold = d->all ? 0xffffffffu : static_cast<unsigned>(words + 0.5);
    d->scale = d->all ? 0.0f : static_cast<float>(1.0 / (1.0 - p));
    return true;
}

#ifdef __CUDACC__
template <class T>
__device__ __forceinline__ float to_float(T v) {
    if constexpr (std::is_same_v<T, float>) return v;
    else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
    else return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T from_float(float v) {
    if constexpr (std::is_same_v<T, float>) return v;
    else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}
template <class T>
__device__ __forceinline__ float rounded(float v) {
    return to_float(from_float<T>(v));
}

// A parameter of a layer: 32 bits, or the type of the activations
template <class T>
__device__ __forceinline__ float param_at(const void* p, bool wide, long long i) {
    return wide ? static_cast<const float*>(p)[i] : to_float(static_cast<const T*>(p)[i]);
}
template <class T>
__device__ __forceinline__ void set_param(void* p, bool wide, long long i, float v) {
    if (wide) static_cast<float*>(p)[i] = v;
    else static_cast<T*>(p)[i] = from_float<T>(v);
}

// ---- the generator ---------------------------------------------------------------------------------------------------------
// Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011): four words
// from a 64-bit key and a 128-bit counter, here the seed and (block, offset).  Element i takes word i % 4 of block i / 4, so the
// mask is a function of seed, offset and the element's place alone: the backward pass makes it again, whatever its launch.
struct Generator {
    unsigned key0, key1, c2, c3;
};
__device__ __forceinline__ Generator generator_of(const DropoutArgs& d) {
    const unsigned long long seed = d.state ? d.state[0] : d.seed, offset = d.offset + (d.state ? d.state[1] : 0ull);
    return Generator{static_cast<unsigned>(seed), static_cast<unsigned>(seed >> 32), static_cast<unsigned>(offset),
                     static_cast<unsigned>(offset >> 32)};
}
__device__ __forceinline__ uint4 random_words(const Generator& g, unsigned long long block) {
    unsigned c0 = static_cast<unsigned>(block), c1 = static_cast<unsigned>(block >> 32), c2 = g.c2, c3 = g.c3;
    unsigned k0 = g.key0, k1 = g.key1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = 0xD2511F53ull * c0, b = 0xCD9E8D57ull * c2;
        c0 = static_cast<unsigned>(b >> 32) ^ c1 ^ k0;
        c1 = static_cast<unsigned>(b);
        c2 = static_cast<unsigned>(a >> 32) ^ c3 ^ k1;
        c3 = static_cast<unsigned>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ unsigned random_word(const Generator& g, unsigned long long i) {
    const uint4 w = random_words(g, i >> 2);
    const unsigned lane = static_cast<unsigned>(i) & 3u;
    return lane == 0 ? w.x : lane == 1 ? w.y : lane == 2 ? w.z : w.w;
}
// (the product is rounded by itself, so that every path and every neighbouring addition gives the same bits)
__device__ __forceinline__ float dropped(const DropoutArgs& d, unsigned word, float v) {
    return word >= d.threshold && !d.all ? __fmul_rn(v, d.scale) : 0.0f;
}

// ---- sums over a block of whole warps ------------------------------------------------------------------------------------------
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Sum over the block's threads in a fixed order, for all of them; `slots` holds a float per warp.
__device__ __forceinline__ float block_sum(float v, float* slots) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (unsigned w = 0; w < blockDim.x >> 5; ++w) s += slots[w];
    return s;
}

// ---- rows as 8-bit integers ----------------------------------------------------------------------------------------------------
// The bits of |v|: their order is that of the magnitudes, with infinity above all numbers and what is not a number above that.
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// A row's step: its largest magnitude is 127 steps, and no step is below the smallest normal number, so that its reciprocal is
// finite; a row with a value that is not finite has such a step, and all its products are not-a-number.
__device__ __forceinline__ float step_of(unsigned largest) {
    const float s = __fdiv_rn(__uint_as_float(largest), 127.0f);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
// The nearest integer number of steps, ties to even: |v| <= 127 step (1 + 2^-24), so it has 8 bits; 0 for what is not a number
__device__ __forceinline__ int steps(float v, float inverse) { return __float2int_rn(__fmul_rn(v, inverse)); }
#endif  // __CUDACC__

}  // namespace ldn
