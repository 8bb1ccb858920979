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
// Columns of a row and outputs of a product, at most: a column plus a grid's or a tile's size is still an int
constexpr int kMostColumns = 0x7fffffff - (1 << 22);
inline bool row_fits(int C) { return C > 0 && C <= kMostColumns; }
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
//
// An integer product of two words takes the integer pipe for two clocks a warp, as an exclusive or does (84 million words take 50 us
// at best; 16-bit dropout takes 90, memory 51).  So what does not depend on the block is made once: the round
// keys, and of the first two rounds all but one product each, as the block's high word is 0 for the first 2^34 elements.
struct Generator {
    unsigned key[20], c2, c3;
    unsigned first, second, third, fourth;  // of rounds 1 and 2, for blocks below 2^32
};
// (low, high) word of a product
__device__ __forceinline__ uint2 wide_product(unsigned a, unsigned b) {
    uint2 r;
    asm("{\n\t.reg .u64 t;\n\tmul.wide.u32 t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}" : "=r"(r.x), "=r"(r.y) : "r"(a), "r"(b));
    return r;
}
constexpr unsigned kPhilox0 = 0xD2511F53u, kPhilox1 = 0xCD9E8D57u;
// One round: (c0, c1, c2, c3) with the keys k0 and k1
__device__ __forceinline__ void philox_round(unsigned& c0, unsigned& c1, unsigned& c2, unsigned& c3, unsigned k0, unsigned k1) {
    const uint2 a = wide_product(c0, kPhilox0), b = wide_product(c2, kPhilox1);
    c0 = b.y ^ c1 ^ k0;
    c1 = b.x;
    c2 = a.y ^ c3 ^ k1;
    c3 = a.x;
}
__device__ __forceinline__ Generator generator_of(const DropoutArgs& d) {
    const unsigned long long seed = d.state ? d.state[0] : d.seed, offset = d.offset + (d.state ? d.state[1] : 0ull);
    Generator g;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        g.key[2 * r] = static_cast<unsigned>(seed) + r * 0x9E3779B9u;
        g.key[2 * r + 1] = static_cast<unsigned>(seed >> 32) + r * 0xBB67AE85u;
        asm volatile("" : "+r"(g.key[2 * r]), "+r"(g.key[2 * r + 1]));  // (kept, not made again for every block)
    }
    g.c2 = static_cast<unsigned>(offset);
    g.c3 = static_cast<unsigned>(offset >> 32);
    const uint2 b1 = wide_product(g.c2, kPhilox1), a2 = wide_product(b1.y ^ g.key[0], kPhilox0);
    g.first = g.c3 ^ g.key[1];
    g.second = b1.x ^ g.key[2];
    g.third = a2.y ^ g.key[3];
    g.fourth = a2.x;
    return g;
}
static __device__ __noinline__ uint4 random_words_beyond(unsigned long long seed_low_high, unsigned long long offset, unsigned long long block) {
    unsigned c0 = static_cast<unsigned>(block), c1 = static_cast<unsigned>(block >> 32), c2 = static_cast<unsigned>(offset),
             c3 = static_cast<unsigned>(offset >> 32), k0 = static_cast<unsigned>(seed_low_high), k1 = static_cast<unsigned>(seed_low_high >> 32);
    for (int r = 0; r < 10; ++r) {
        philox_round(c0, c1, c2, c3, k0, k1);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint4 random_words(const Generator& g, unsigned long long block) {
    if (block >> 32)
        return random_words_beyond(g.key[0] | static_cast<unsigned long long>(g.key[1]) << 32,
                                   g.c2 | static_cast<unsigned long long>(g.c3) << 32, block);
    const uint2 a1 = wide_product(static_cast<unsigned>(block), kPhilox0), b2 = wide_product(a1.y ^ g.first, kPhilox1);
    unsigned c0 = b2.y ^ g.second, c1 = b2.x, c2 = a1.x ^ g.third, c3 = g.fourth;
#pragma unroll
    for (int r = 2; r < 10; ++r) philox_round(c0, c1, c2, c3, g.key[2 * r], g.key[2 * r + 1]);
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

// The same for 2 N neighbouring elements from `at` on, a multiple of four (2 N is one, too)
template <int N>
__device__ __forceinline__ void drop_piece(const DropoutArgs& d, const Generator& gen, long long at, float2 (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const uint4 w = random_words(gen, static_cast<unsigned long long>(at + 2 * e) >> 2);
        v[e] = make_float2(dropped(d, w.x, v[e].x), dropped(d, w.y, v[e].y));
        v[e + 1] = make_float2(dropped(d, w.z, v[e + 1].x), dropped(d, w.w, v[e + 1].y));
    }
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
// finite; a row with a value that is not finite has a step that is not a number, and so are all its products
__device__ __forceinline__ float step_of(unsigned largest) {
    if (largest >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
    const float s = __fdiv_rn(__uint_as_float(largest), 127.0f);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
// The nearest integer number of steps, ties to even: |v| <= 127 step (1 + 2^-24), so it has 8 bits (any 8 for what is not a number)
__device__ __forceinline__ int steps(float v, float inverse) { return __float2int_rn(__fmul_rn(v, inverse)); }
// The product of two values with one, rounded (the compiler's packed product may join an addition behind it)
__device__ __forceinline__ float2 rounded_product(float2 v, float s) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmul.rn.f32x2 c, a, b;\n\tmov.b64 {%0, %1}, c;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(v.x), "f"(v.y), "f"(s));
    return r;
}
// The same of four values as bytes: 1.5 2^23 more, the nearest integer is what a number's last bits hold
__device__ __forceinline__ unsigned steps4(float2 a, float2 b, float inverse) {
    a = rounded_product(a, inverse);
    b = rounded_product(b, inverse);
    constexpr float kMagic = 12582912.0f;
    return __byte_perm(__byte_perm(__float_as_uint(__fadd_rn(a.x, kMagic)), __float_as_uint(__fadd_rn(a.y, kMagic)), 0x0040),
                       __byte_perm(__float_as_uint(__fadd_rn(b.x, kMagic)), __float_as_uint(__fadd_rn(b.y, kMagic)), 0x0040), 0x5410);
}
// Largest of two magnitudes, or of one and two values' magnitudes; what is not a number wins
__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float larger(float top, float2 v) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(top), "f"(fabsf(v.x)), "f"(fabsf(v.y)));
    return r;
}
#endif  // __CUDACC__

}  // namespace ldn
