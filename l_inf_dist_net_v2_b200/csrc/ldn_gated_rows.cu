// The gated projection of a handful of rows: the weights are read once and the products are made where they arrive.
//
// Bound by memory: 2 H K elements of the weights.  A block has some outputs, and its threads share their terms in pieces of 16 bytes, so
// that every output's two weight rows are under way at once in whole lines; the rows themselves come from the first-level cache.
// 1, 5120 -> 5120 bf16: 20.2 us, 5.2 TB/s; 1, 5120 -> 2048 float32: 16.7 us, 5.0; 8, 5120 -> 5120 float32: 69 us, 3.0.
#include "ldn_gated.cuh"

namespace ldn {
namespace {

constexpr int kFewThreads = 128;

// A piece of eight elements, `there` of them in the row
template <class T>
__device__ __forceinline__ void piece(const T* p, bool whole, int there, float (&v)[8]) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 raw = *reinterpret_cast<const uint4*>(p);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = to_float(e[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < there ? to_float(p[j]) : 0.0f;
    }
}

// (weights are read once: they leave the first-level cache to the rows)
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <class T>
__device__ __forceinline__ void unpack8(const uint4 (&raw)[sizeof(T) / 2], float (&v)[8]) {
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(e[j]);
}

template <class T, int ROWS, int OUTPUTS>
__global__ void __launch_bounds__(kFewThreads) gated_few_kernel(const __grid_constant__ GatedArgs a, bool aligned) {
    stream_order_begin();
    __shared__ float sums[kFewThreads / 32][2 * OUTPUTS][ROWS];
    const int h0 = blockIdx.x * OUTPUTS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float acc[2 * OUTPUTS][ROWS] = {};
    const T* w[2 * OUTPUTS];
#pragma unroll
    for (int o = 0; o < OUTPUTS; ++o) {
        const long long h = h0 + o < a.H ? h0 + o : a.H - 1;
        w[2 * o] = static_cast<const T*>(a.w_gate) + h * a.pitch_gate;
        w[2 * o + 1] = static_cast<const T*>(a.w_up) + h * a.pitch_up;
    }
    auto add = [&](const float (&wv)[2 * OUTPUTS][8], int c, bool whole) {
#pragma unroll
        for (int t = 0; t < ROWS; ++t) {
            float xv[8];
            const long long row = t < a.T ? t : a.T - 1;
            piece(static_cast<const T*>(a.x) + row * a.pitch_x + c, whole, a.K - c, xv);
#pragma unroll
            for (int o = 0; o < 2 * OUTPUTS; ++o)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[o][t] = fmaf(wv[o][j], xv[j], acc[o][t]);
        }
    };
    // Whole pieces, kAhead of each weight row under way at a time (two at a time, and through the cache: 26.6 us for 1, 5120 -> 5120 bf16)
    constexpr int kStep = kFewThreads * 8, kAhead = sizeof(T) * OUTPUTS >= 8 ? 2 : 4, kWords = sizeof(T) / 2;
    const int whole_end = aligned ? a.K / 8 * 8 : 0;
    int c = threadIdx.x * 8;
    for (; c < whole_end; c += kAhead * kStep) {
        uint4 raw[kAhead][2 * OUTPUTS][kWords];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c + u * kStep < whole_end)
#pragma unroll
                for (int o = 0; o < 2 * OUTPUTS; ++o)
#pragma unroll
                    for (int i = 0; i < kWords; ++i) raw[u][o][i] = load_once(reinterpret_cast<const uint4*>(w[o] + c + u * kStep) + i);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c + u * kStep < whole_end) {
                float wv[2 * OUTPUTS][8];
#pragma unroll
                for (int o = 0; o < 2 * OUTPUTS; ++o) unpack8<T>(raw[u][o], wv[o]);
                add(wv, c + u * kStep, true);
            }
    }
    // what is left of a row, or all of it where rows are not aligned
    for (c = whole_end + threadIdx.x * 8; c < a.K; c += kStep) {
        float wv[2 * OUTPUTS][8];
#pragma unroll
        for (int o = 0; o < 2 * OUTPUTS; ++o) piece(w[o] + c, false, a.K - c, wv[o]);
        add(wv, c, false);
    }
#pragma unroll
    for (int o = 0; o < 2 * OUTPUTS; ++o)
#pragma unroll
        for (int t = 0; t < ROWS; ++t) {
            const float s = warp_sum(acc[o][t]);
            if (lane == 0) sums[warp][o][t] = s;
        }
    __syncthreads();
    if (threadIdx.x < OUTPUTS * ROWS) {
        const int o = threadIdx.x / ROWS, t = threadIdx.x % ROWS, h = h0 + o;
        if (h < a.H && t < a.T) {
            float g[1] = {0.0f}, u = 0.0f;
#pragma unroll
            for (int i = 0; i < kFewThreads / 32; ++i) {
                g[0] += sums[i][2 * o][t];
                u += sums[i][2 * o + 1][t];
            }
            if (a.b_gate) g[0] += param_at<T>(a.b_gate, a.wide, h);
            if (a.b_up) u += param_at<T>(a.b_up, a.wide, h);
            if (a.g) {
                a.g[t * a.pitch_saved + h] = g[0];
                a.u[t * a.pitch_saved + h] = u;
            }
            activate(g, a.activation);
            static_cast<T*>(a.y)[static_cast<long long>(t) * a.H + h] = from_float<T>(g[0] * u);
        }
    }
}

// (a block's outputs, 1 / 2: 1 row 5120 -> 5120 bf16 21.5 / 20.2 us; 128 threads, 64: 21.0, 256: 23.2 with one output each)
constexpr int kOutputs = 2;
template <class T, int ROWS>
int launch(const GatedArgs& a, bool aligned, cudaStream_t st) {
    return launch_after(gated_few_kernel<T, ROWS, kOutputs>, (a.H + kOutputs - 1) / kOutputs, kFewThreads, 0, st, a, aligned);
}
bool at_16(const void* p, long long pitch, long long rows, int size) {
    return ((reinterpret_cast<uintptr_t>(p) | (rows > 1 ? static_cast<uintptr_t>(pitch) * size : 0)) & 15u) == 0;
}
bool all_at_16(const GatedArgs& a, int size) {
    return at_16(a.x, a.pitch_x, a.T, size) && at_16(a.w_gate, a.pitch_gate, a.H, size) && at_16(a.w_up, a.pitch_up, a.H, size);
}

}  // namespace

// Where the tensor cores take longer.  5120 -> 5120, us, here / there: bf16 1 row 20 / 29, 2 rows 22 / 29, 4 rows 33 / 29; one row of 5119, whose
// weights would be copied, 37; float32, whose weights would be written as three images, 8 rows 69 / 182.
bool gated_is_few(const GatedArgs& a, int type) {
    return a.T <= (type == LDN_F32 ? 16 : all_at_16(a, size_of(type)) ? 2 : 4);
}

int launch_gated_few(const GatedArgs& a, int type, cudaStream_t st) {
    const bool aligned = all_at_16(a, size_of(type));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (a.T <= 1) return launch<T, 1>(a, aligned, st);
        if (a.T <= 2) return launch<T, 2>(a, aligned, st);
        if constexpr (sizeof(T) == 4) {
            if (a.T > 8) return launch<T, 16>(a, aligned, st);
            if (a.T > 4) return launch<T, 8>(a, aligned, st);
        }
        return launch<T, 4>(a, aligned, st);
    });
}

}  // namespace ldn
