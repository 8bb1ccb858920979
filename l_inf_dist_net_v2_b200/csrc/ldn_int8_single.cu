// The integer product of one to four tokens: the weight is read once and nothing else counts, so it is one launch.  A block quantises
// the tokens for itself, with its first pieces of the weight already under way, and takes every gridDim-th output: pieces of a row of the
// weight of up to 1024 terms are dealt out to its warps (whole rows would leave a third of them idle at 35 outputs per SM), four
// products per instruction and token, and their sums meet in shared memory as integers, in which no order shows.
//
// 5120 -> 5120 in bf16, from memory 14.3 us between events (the first load waits for the kernel in front); weight in L2, us, one launch / quantising and tiles on the tensor cores: one token 7.3 / 9.8, two 9.0 / 9.9,
// four 12.3 / 10.2 (4 x 1000 x 3000: 5.8 / 8); as whole rows with scalar loads one token took 9.2.
#include "ldn_int8.cuh"

namespace ldn {
namespace {

constexpr int kSingleThreads = 512, kSingleWarps = kSingleThreads / 32;
constexpr int kPieceTerms = 1024;    // two 16-byte loads per lane
constexpr int kPiecesAhead = 4;
constexpr int kMostRows = 1024;      // of a block
constexpr int kMostTokenBytes = 128 << 10;

struct SingleArgs {
    ProductArgs product;
    const void* x;      // rows in floating point, or null: product.q and product.scale
    long long pitch;
    int out_type;
    int rows;           // outputs per block, at most
    bool vectors;       // four elements of x from a multiple of four on are one load
};

template <class T, int TOKENS>
__global__ void __launch_bounds__(kSingleThreads, 1) product_single_kernel(SingleArgs s) {
    stream_order_begin();
    extern __shared__ uint4 tokens[];  // [token][padded terms] bytes, then [output][token] sums
    __shared__ unsigned largest[TOKENS];
    __shared__ float scale[TOKENS];
    const ProductArgs& a = s.product;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pieces = (a.K + kPieceTerms - 1) / kPieceTerms, padded = pieces * kPieceTerms;
    signed char* q = reinterpret_cast<signed char*>(tokens);
    int* sums = reinterpret_cast<int*>(q + TOKENS * padded);
    const int outputs = (a.N - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    // piece and output of a warp's tasks, from one to the next
    struct Task {
        int out, piece;
    };
    const int step_out = kSingleWarps / pieces, step_piece = kSingleWarps % pieces;
    auto next = [&](Task& t) {
        t.out += step_out;
        t.piece += step_piece;
        if (t.piece >= pieces) {
            t.piece -= pieces;
            ++t.out;
        }
    };
    auto fetch = [&](const Task& t, uint4 (&w)[2]) {
        const int k0 = t.piece * kPieceTerms + lane * 16;
        const long long n = blockIdx.x + static_cast<long long>(t.out) * gridDim.x;
        const signed char* row = a.w + n * a.pitch_w;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = k0 + h * 512;
            w[h] = make_uint4(0u, 0u, 0u, 0u);
            if (t.out >= outputs || k >= a.K) continue;
            // (the 16 bytes at a row's end reach into its padding; the last row may have none)
            if (k + 16 <= a.K || n + 1 < a.N) {
                w[h] = __ldg(reinterpret_cast<const uint4*>(row + k));
            } else {
                unsigned v[4] = {};
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (k + e < a.K) v[e / 4] |= static_cast<unsigned>(static_cast<unsigned char>(row[k + e])) << 8 * (e % 4);
                w[h] = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
    };
    uint4 ahead[kPiecesAhead][2];
    Task to_fetch = {warp / pieces, warp % pieces}, to_add = to_fetch;
#pragma unroll
    for (int i = 0; i < kPiecesAhead; ++i, next(to_fetch)) fetch(to_fetch, ahead[i]);

    for (int i = threadIdx.x; i < outputs * TOKENS; i += kSingleThreads) sums[i] = 0;
    constexpr int kShare = kSingleThreads / TOKENS;  // threads per token
    const int m = threadIdx.x / kShare, t = threadIdx.x % kShare;
    if constexpr (std::is_same_v<T, signed char>) {
        if (t == 0) scale[m] = m < a.M ? a.scale[m] : 0.0f;
        for (int k = t; k < padded; k += kShare) q[m * padded + k] = m < a.M && k < a.K ? a.q[m * a.pitch_q + k] : 0;
        __syncthreads();
    } else {
        if (threadIdx.x < TOKENS) largest[threadIdx.x] = 0u;
        __syncthreads();
        const T* row = static_cast<const T*>(s.x) + (m < a.M ? m : 0) * s.pitch;
        const int K = m < a.M ? a.K : 0;
        auto four = [&](int k) {
            float v[4];
            if (s.vectors && k + 4 <= K) {
                if constexpr (sizeof(T) == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(row + k);
                    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
                } else {
                    T h[4];
                    *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(row + k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = to_float(h[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = k + e < K ? to_float(row[k + e]) : 0.0f;
            }
            return make_float4(v[0], v[1], v[2], v[3]);
        };
        // (the first three turns' values stay in registers for the second pass)
        constexpr int kHeld = 3;
        float4 held[kHeld];
        float top = 0.0f;
        auto take = [&](const float4& v) { top = larger(larger(top, make_float2(v.x, v.y)), make_float2(v.z, v.w)); };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) held[i] = four(4 * (t + i * kShare));
#pragma unroll
        for (int i = 0; i < kHeld; ++i) take(held[i]);
        for (int k = 4 * (t + kHeld * kShare); k < K; k += 4 * kShare) take(four(k));
        const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if (lane == 0) atomicMax(&largest[m], bits);
        __syncthreads();
        const float size = step_of(largest[m]), inverse = 1.0f / size;
        if (t == 0) scale[m] = size;
        auto put = [&](int k, const float4& v) {
            *reinterpret_cast<unsigned*>(q + m * padded + k) = steps4(make_float2(v.x, v.y), make_float2(v.z, v.w), inverse);
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (4 * (t + i * kShare) < padded) put(4 * (t + i * kShare), held[i]);
        for (int k = 4 * (t + kHeld * kShare); k < padded; k += 4 * kShare) put(k, four(k));
        __syncthreads();
    }

    while (to_add.out < outputs) {
#pragma unroll
        for (int i = 0; i < kPiecesAhead; ++i) {
            if (to_add.out < outputs) {
                const int k = to_add.piece * kPieceTerms + lane * 16;
                int sum[TOKENS];
#pragma unroll
                for (int c = 0; c < TOKENS; ++c) {
                    sum[c] = 0;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 v = *reinterpret_cast<const uint4*>(q + c * padded + k + h * 512);
                        sum[c] = __dp4a(static_cast<int>(v.x), static_cast<int>(ahead[i][h].x), sum[c]);
                        sum[c] = __dp4a(static_cast<int>(v.y), static_cast<int>(ahead[i][h].y), sum[c]);
                        sum[c] = __dp4a(static_cast<int>(v.z), static_cast<int>(ahead[i][h].z), sum[c]);
                        sum[c] = __dp4a(static_cast<int>(v.w), static_cast<int>(ahead[i][h].w), sum[c]);
                    }
                }
                fetch(to_fetch, ahead[i]);
#pragma unroll
                for (int c = 0; c < TOKENS; ++c) {
                    sum[c] = __reduce_add_sync(0xffffffffu, sum[c]);
                    if (lane == 0) atomicAdd(&sums[to_add.out * TOKENS + c], sum[c]);
                }
                next(to_fetch);
                next(to_add);
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < outputs * TOKENS; i += kSingleThreads) {
        const int c = i % TOKENS, n = static_cast<int>(blockIdx.x) + i / TOKENS * static_cast<int>(gridDim.x);
        if (c >= a.M) continue;
        const float v = product_value(sums[i], scale[c], a.w_scale[n], a.bias ? a.bias[n] : 0.0f, a.activation);
        const long long at = c * static_cast<long long>(a.N) + n;
        if (s.out_type == LDN_F32) static_cast<float*>(a.out)[at] = v;
        else if (s.out_type == LDN_F16) static_cast<__half*>(a.out)[at] = from_float<__half>(v);
        else static_cast<__nv_bfloat16*>(a.out)[at] = from_float<__nv_bfloat16>(v);
    }
}

template <class T, int TOKENS>
int launch(SingleArgs s, const DeviceCtx* ctx, cudaStream_t st) {
    static OncePerDevice once;
    constexpr int kMostSmem = kMostTokenBytes + kMostRows * TOKENS * 4;
    const int r = once([] { return allow_smem(product_single_kernel<T, TOKENS>, kMostSmem); });
    if (r != kOk) return r;
    int grid = s.product.N < ctx->sm_count ? s.product.N : ctx->sm_count;
    if ((s.product.N + grid - 1) / grid > kMostRows) grid = (s.product.N + kMostRows - 1) / kMostRows;
    s.rows = (s.product.N + grid - 1) / grid;
    const size_t padded = static_cast<size_t>(s.product.K + kPieceTerms - 1) / kPieceTerms * kPieceTerms;
    return launch_after(product_single_kernel<T, TOKENS>, grid, kSingleThreads, TOKENS * (padded + s.rows * sizeof(int)), st, s);
}
template <class T>
int launch(const SingleArgs& s, const DeviceCtx* ctx, cudaStream_t st) {
    return s.product.M == 1 ? launch<T, 1>(s, ctx, st) : s.product.M == 2 ? launch<T, 2>(s, ctx, st) : launch<T, 4>(s, ctx, st);
}

}  // namespace

bool product_is_single(const ProductArgs& a) {
    const long long padded = (a.K + kPieceTerms - 1LL) / kPieceTerms * kPieceTerms, tokens = a.M <= 2 ? a.M : 4;
    // (three and four tokens: up to where the tensor cores' fixed costs are made up for, about 8 MB of weight)
    if (a.M > 2 && static_cast<long long>(a.N) * a.K > 8 << 20) return false;
    return a.M <= 4 && tokens * padded <= kMostTokenBytes && a.pitch_w % 16 == 0 && (reinterpret_cast<uintptr_t>(a.w) & 15u) == 0;
}

int launch_product_single(const ProductArgs& a, const void* x, long long pitch, int x_type, int out_type, const DeviceCtx* ctx,
                          cudaStream_t st) {
    const int four = x ? 4 * size_of(x_type) : 4;
    const SingleArgs s = {a, x, pitch, out_type, 0, reinterpret_cast<uintptr_t>(x) % four == 0 && pitch % 4 == 0};
    if (!x) return launch<signed char>(s, ctx, st);
    return with_type(x_type, [&](auto t) { return launch<decltype(t)>(s, ctx, st); });
}

}  // namespace ldn
