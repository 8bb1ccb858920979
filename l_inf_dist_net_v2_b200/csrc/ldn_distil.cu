// Distillation from a teacher's top logits, mixed with the cross-entropy of labels, and its gradient:
//     p = softmax(t / tau) over the entries of a row's list,   q = softmax(x / tau) over all classes,
//     loss = part tau^2 sum p (log p - log q) + mix (log sum e^x - x[label]),
//     dx = up (part tau (q - p) + mix (softmax(x) - [label])).
// A list's entry below 0 is absent, a row without entries has no first term, a row with a label below 0 no second; an index beyond the
// classes makes the row's loss and gradient not-a-numbers.
//
// Bound by memory: forward x once (the largest logit and both sums come of one pass, the sums rescaled when a larger logit comes),
// backward x and dx once: the gradient of a row is written whole as if it had no list, and then at the list's classes.
#include "ldn_head.cuh"
#include "ldn_tensor.cuh"

namespace ldn {
namespace {

constexpr int kDistilThreads = 256, kDistilWarps = kDistilThreads / 32;
constexpr int kMostEntries = 1024;
constexpr int kMostRanks = 8;  // CTAs of a cluster that share a row
constexpr float kLog2e = 1.4426950408889634f;

struct DistilArgs {
    const void* x;
    long long pitch, rows;
    int V;
    const void* values;  // [rows][k]
    int value_type, k;
    const long long* indices;  // [rows][k]
    const long long* targets;  // [rows], may be null
    float tau, part, mix;
    float* losses;  // [rows]
    float* stats;   // [5][rows]: largest logit, 1 / sums at tau and at 1, the list's largest value / tau, 1 / its sum
    // backward
    const float* up;
    int up_step;      // 0: one number for all rows
    float up_scale;
    void* grad;  // [rows][V]
};

__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float largest_of(float a, float b) {  // (what is not a number wins)
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float minus_infinity() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float not_a_number() { return __int_as_float(0x7fffffff); }

// Largest logit so far, and the sums of e^((x - largest) / tau) and of e^(x - largest)
struct Sums {
    float m, s, s1;
    __device__ __forceinline__ void join(float om, float os, float os1, float c, float c1) {
        const float top = largest_of(m, om);
        const float a = m == top ? 1.0f : exp2_fast((m - top) * c), b = om == top ? 1.0f : exp2_fast((om - top) * c);
        const float a1 = m == top ? 1.0f : exp2_fast((m - top) * c1), b1 = om == top ? 1.0f : exp2_fast((om - top) * c1);
        s = s * a + os * b;
        s1 = s1 * a1 + os1 * b1;
        m = top;
    }
    __device__ __forceinline__ void over_lanes(int lanes, float c, float c1) {
        for (int d = lanes >> 1; d > 0; d >>= 1)
            join(__shfl_xor_sync(0xffffffffu, m, d), __shfl_xor_sync(0xffffffffu, s, d), __shfl_xor_sync(0xffffffffu, s1, d), c, c1);
    }
};

// A row in pieces of 16 bytes at memory's boundaries: piece j has the elements j N - shift ..
template <class T>
struct Pieces {
    static constexpr int N = 16 / sizeof(T);
    const T* row;
    int V, shift, count;
    __device__ __forceinline__ Pieces(const T* r, int v) : row(r), V(v) {
        shift = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
        count = static_cast<int>((static_cast<long long>(v) + shift + N - 1) / N);
    }
    __device__ __forceinline__ int first(int j) const { return j * N - shift; }
    __device__ __forceinline__ bool whole(int j) const { return first(j) >= 0 && first(j) + N <= V; }
    __device__ __forceinline__ uint4 load(int j) const { return *reinterpret_cast<const uint4*>(row + first(j)); }
    static __device__ __forceinline__ void unpack(uint4 raw, float (&v)[N]) {
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(e[i]);
    }
    // a piece at either end, `none` outside the row
    __device__ __forceinline__ void edge(int j, float none, float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = first(j) + i;
            v[i] = static_cast<unsigned>(c) < static_cast<unsigned>(V) ? to_float(row[c]) : none;
        }
    }
};

template <int N>
__device__ __forceinline__ void add_values(Sums& a, const float (&v)[N], float c, float c1, bool second) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = largest_of(top, v[i]);
    if (!(top <= a.m)) {
        a.s *= exp2_fast((a.m - top) * c);
        a.s1 *= exp2_fast((a.m - top) * c1);
        a.m = top;
    }
    if (a.m == minus_infinity()) return;
#pragma unroll
    for (int i = 0; i < N; ++i) a.s += exp2_fast((v[i] - a.m) * c);
    if (second) {
#pragma unroll
        for (int i = 0; i < N; ++i) a.s1 += exp2_fast((v[i] - a.m) * c1);
    }
}

__device__ __forceinline__ float value_at(const DistilArgs& a, long long i) {
    return a.value_type == LDN_F32 ? static_cast<const float*>(a.values)[i]
         : a.value_type == LDN_F16 ? __half2float(static_cast<const __half*>(a.values)[i])
                                   : __bfloat162float(static_cast<const __nv_bfloat16*>(a.values)[i]);
}

// What a warp makes of a row's sums: its loss, and what the backward pass needs
template <class T>
__device__ __forceinline__ void finish_row(const DistilArgs& a, long long row, const Sums& sums) {
    const int lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(a.x) + row * a.pitch;
    const long long* indices = a.indices + row * a.k;
    const float inv_tau = 1.0f / a.tau;
    bool bad = false;
    float top = minus_infinity();
    for (int j = lane; j < a.k; j += 32) {
        const long long i = indices[j];
        bad = bad || i >= a.V;
        if (i >= 0) top = largest_of(top, value_at(a, row * a.k + j) * inv_tau);
    }
    for (int d = 16; d > 0; d >>= 1) top = largest_of(top, __shfl_xor_sync(0xffffffffu, top, d));
    bad = __any_sync(0xffffffffu, bad);
    float sum = 0.0f;
    const bool some = top != minus_infinity();  // (a list of nothing but minus infinity says nothing)
    if (some)
        for (int j = lane; j < a.k; j += 32)
            if (indices[j] >= 0) sum += expf(value_at(a, row * a.k + j) * inv_tau - top);
    sum = warp_sum(sum);
    const float log_s = logf(sums.s), log_sum = logf(sum), inv_sum = 1.0f / sum;
    float loss = 0.0f;
    if (some && !bad) {
        for (int j = lane; j < a.k; j += 32) {
            const long long i = indices[j];
            if (i < 0) continue;
            const float t = value_at(a, row * a.k + j) * inv_tau - top, p = expf(t) * inv_sum;
            // log p - log q, each relative to its largest
            if (p != 0.0f) loss += p * ((t - log_sum) - ((to_float(x[i]) - sums.m) * inv_tau - log_s));
        }
        loss = warp_sum(loss) * (a.part * a.tau * a.tau);
    }
    float s1 = sums.s1;
    if (a.tau == 1.0f) s1 = sums.s;
    if (a.targets) {
        const long long target = a.targets[row];
        bad = bad || target >= a.V;
        if (target >= 0 && !bad) loss += a.mix * (logf(s1) - (to_float(x[target]) - sums.m));
    }
    if (lane == 0) {
        a.losses[row] = bad ? not_a_number() : loss;
        if (a.stats) {
            a.stats[row] = sums.m;
            a.stats[a.rows + row] = bad ? not_a_number() : 1.0f / sums.s;
            a.stats[2 * a.rows + row] = bad ? not_a_number() : 1.0f / s1;
            a.stats[3 * a.rows + row] = top;
            a.stats[4 * a.rows + row] = bad ? not_a_number() : some ? inv_sum : 0.0f;
        }
    }
}

// A row of up to kShort classes: a warp.  Longer ones: a block, or the blocks of a cluster, each with a range of the pieces.
constexpr int kShort = 2048, kAhead = 4;
template <class T>
__device__ __forceinline__ void read_pieces(const Pieces<T>& p, int first, int last, int thread, int threads, const DistilArgs& a, float c,
                                            float c1, bool second, Sums& sums) {
    constexpr int N = Pieces<T>::N;
    int j = first + thread;
    for (; j + (kAhead - 1) * threads < last; j += kAhead * threads) {
        uint4 raw[kAhead];
        const bool whole = p.whole(j) && p.whole(j + (kAhead - 1) * threads);  // (and so are those between)
        if (whole) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) raw[u] = p.load(j + u * threads);
            float v[kAhead * N];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) Pieces<T>::unpack(raw[u], reinterpret_cast<float(&)[N]>(v[u * N]));
            add_values(sums, v, c, c1, second);
        } else {
            for (int u = 0; u < kAhead; ++u) {
                float v[N];
                p.edge(j + u * threads, minus_infinity(), v);
                add_values(sums, v, c, c1, second);
            }
        }
    }
    for (; j < last; j += threads) {
        float v[N];
        if (p.whole(j)) Pieces<T>::unpack(p.load(j), v);
        else p.edge(j, minus_infinity(), v);
        add_values(sums, v, c, c1, second);
    }
}

template <class T>
__global__ void __launch_bounds__(kDistilThreads) distil_short_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    const float c = kLog2e / a.tau, c1 = kLog2e;
    const bool second = a.targets && a.tau != 1.0f;
    for (long long row = static_cast<long long>(blockIdx.x) * kDistilWarps + (threadIdx.x >> 5); row < a.rows;
         row += static_cast<long long>(gridDim.x) * kDistilWarps) {
        const Pieces<T> p(static_cast<const T*>(a.x) + row * a.pitch, a.V);
        Sums sums = {minus_infinity(), 0.0f, 0.0f};
        read_pieces(p, 0, p.count, threadIdx.x & 31, 32, a, c, c1, second, sums);
        __syncwarp();
        sums.over_lanes(32, c, c1);
        finish_row<T>(a, row, sums);
    }
}

template <class T>
__global__ void __launch_bounds__(kDistilThreads) distil_long_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    __shared__ Sums of_warps[kDistilWarps], of_ranks[kMostRanks];
    const float c = kLog2e / a.tau, c1 = kLog2e;
    const bool second = a.targets && a.tau != 1.0f;
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const long long row = blockIdx.x / ranks;
    if (ranks > 1) cluster_barrier();  // (the first CTA is there to be written to)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Pieces<T> p(static_cast<const T*>(a.x) + row * a.pitch, a.V);
    Sums sums = {minus_infinity(), 0.0f, 0.0f};
    read_pieces(p, static_cast<int>(static_cast<long long>(p.count) * rank / ranks), static_cast<int>(static_cast<long long>(p.count) * (rank + 1) / ranks),
                threadIdx.x, kDistilThreads, a, c, c1, second, sums);
    __syncwarp();
    sums.over_lanes(32, c, c1);
    if (lane == 0) of_warps[warp] = sums;
    __syncthreads();
    if (warp == 0) {
        sums = lane < kDistilWarps ? of_warps[lane] : Sums{minus_infinity(), 0.0f, 0.0f};
        sums.over_lanes(32, c, c1);
        if (ranks > 1 && lane == 0) {
            const uint32_t to = in_cta(&of_ranks[rank], 0);
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(sums.m) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(sums.s) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(sums.s1) : "memory");
        }
    }
    if (ranks > 1) {
        __syncthreads();
        cluster_barrier();
        if (rank == 0 && warp == 0) {
            sums = lane < static_cast<int>(ranks) ? of_ranks[lane] : Sums{minus_infinity(), 0.0f, 0.0f};
            sums.over_lanes(32, c, c1);
        }
    }
    if (rank == 0 && warp == 0) finish_row<T>(a, row, sums);
}

// The rows' losses in a fixed order
constexpr int kMeanThreads = 1024;
__global__ void __launch_bounds__(kMeanThreads) distil_mean_kernel(const float* losses, long long rows, float scale, float* out) {
    stream_order_begin();
    __shared__ float slots[kMeanThreads / 32];
    float s[4] = {};
    for (long long i = threadIdx.x; i < rows; i += 4 * kMeanThreads) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * kMeanThreads < rows) s[u] += losses[i + u * kMeanThreads];
    }
    const float all = block_sum((s[0] + s[1]) + (s[2] + s[3]), slots);
    if (threadIdx.x == 0) *out = all * scale;
}

// ---- backward -------------------------------------------------------------------------------------------------------------------------
// What a row's gradient is made of: w e^((x - m) c) + w1 e^((x - m) c1), less the list's and the label's
struct RowGradient {
    float m, w, w1, c, c1;
    bool one, two;
    __device__ __forceinline__ float operator()(float x) const {
        const float d = x - m;
        float v = one ? w * exp2_fast(d * c) : 0.0f;
        if (two) v += w1 * exp2_fast(d * c1);
        return v;
    }
};

template <class T, int THREADS>
__device__ __forceinline__ void gradient_of_row(const DistilArgs& a, long long row, int part, int parts, int thread, long long* index, float* minus) {
    constexpr int N = Pieces<T>::N;
    const T* x = static_cast<const T*>(a.x) + row * a.pitch;
    T* to = static_cast<T*>(a.grad) + row * a.V;
    const float up = a.up[row * a.up_step] * a.up_scale;
    const float inv_sum = a.stats[4 * a.rows + row], top = a.stats[3 * a.rows + row], inv_tau = 1.0f / a.tau;
    const long long target = a.targets ? a.targets[row] : -1;
    const bool list = inv_sum != 0.0f, label = target >= 0;  // (a list that is not a number is there)
    const float by_list = list ? up * a.part * a.tau : 0.0f, by_label = label ? up * a.mix : 0.0f;
    RowGradient g;
    g.m = a.stats[row];
    g.c = kLog2e * inv_tau;
    g.c1 = kLog2e;
    g.one = list;
    g.two = label;
    g.w = by_list * a.stats[a.rows + row];
    g.w1 = by_label * a.stats[2 * a.rows + row];
    if (a.tau == 1.0f && label) {  // (one and the same softmax)
        g.w = (list ? g.w : 0.0f) + g.w1;
        g.one = true;
        g.two = false;
    }
    const Pieces<T> p(x, a.V);
    const int first = static_cast<int>(static_cast<long long>(p.count) * part / parts), last = static_cast<int>(static_cast<long long>(p.count) * (part + 1) / parts);
    const int begin = p.first(first) > 0 ? p.first(first) : 0, end = p.first(last) < a.V ? p.first(last) : a.V;
    // the list, and the label behind it
    for (int j = thread; j <= a.k; j += THREADS) {
        const long long i = j < a.k ? a.indices[row * a.k + j] : target;
        index[j] = i;
        minus[j] = j == a.k ? by_label : i >= 0 && list ? by_list * (expf(value_at(a, row * a.k + j) * inv_tau - top) * inv_sum) : 0.0f;
    }
    const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(to)) & 15u) == 0;
    constexpr int kRow = 2;
    if (same) {
        for (int j0 = first + thread; j0 < last; j0 += kRow * THREADS) {
            uint4 raw[kRow];
#pragma unroll
            for (int u = 0; u < kRow; ++u)
                if (j0 + u * THREADS < last && p.whole(j0 + u * THREADS)) raw[u] = p.load(j0 + u * THREADS);
#pragma unroll
            for (int u = 0; u < kRow; ++u) {
                const int j = j0 + u * THREADS;
                if (j >= last) continue;
                if (p.whole(j)) {
                    float v[N];
                    Pieces<T>::unpack(raw[u], v);
                    T e[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) e[i] = from_float<T>(g(v[i]));
                    *reinterpret_cast<uint4*>(to + p.first(j)) = *reinterpret_cast<const uint4*>(e);
                } else {
                    for (int i = 0; i < N; ++i) {
                        const int c = p.first(j) + i;
                        if (static_cast<unsigned>(c) < static_cast<unsigned>(a.V)) to[c] = from_float<T>(g(to_float(x[c])));
                    }
                }
            }
        }
    } else {
        for (int c = begin + thread; c < end; c += THREADS) to[c] = from_float<T>(g(to_float(x[c])));
    }
    if constexpr (THREADS == 32) __syncwarp();
    else __syncthreads();
    // the list's classes once more: the first entry of a class writes what all its entries take off
    for (int j = thread; j <= a.k; j += THREADS) {
        const long long i = index[j];
        if (i < begin || i >= end) continue;
        float off = 0.0f;
        bool own = true;
        for (int o = 0; o <= a.k; ++o)
            if (index[o] == i) {
                own = own && o >= j;
                off += minus[o];
            }
        if (own) to[i] = from_float<T>(g(to_float(x[i])) - off);
    }
    if constexpr (THREADS == 32) __syncwarp();
}

template <class T>
__global__ void __launch_bounds__(kDistilThreads) distil_grad_short_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    extern __shared__ long long list[];  // [warp][k + 1], then as many floats
    const int warp = threadIdx.x >> 5;
    float* minus = reinterpret_cast<float*>(list + kDistilWarps * (a.k + 1));
    for (long long row = static_cast<long long>(blockIdx.x) * kDistilWarps + warp; row < a.rows; row += static_cast<long long>(gridDim.x) * kDistilWarps)
        gradient_of_row<T, 32>(a, row, 0, 1, threadIdx.x & 31, list + warp * (a.k + 1), minus + warp * (a.k + 1));
}
template <class T>
__global__ void __launch_bounds__(kDistilThreads) distil_grad_long_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    extern __shared__ long long list[];
    const int parts = gridDim.y;
    gradient_of_row<T, kDistilThreads>(a, blockIdx.x, blockIdx.y, parts, threadIdx.x, list, reinterpret_cast<float*>(list + a.k + 1));
}

bool distil_fits(long long rows, int V, int type, int value_type, int k, float tau) {
    return rows >= 0 && rows <= kMostColumns && row_fits(V) && known_type(type) && known_type(value_type) && k >= 1 && k <= kMostEntries &&
           tau > 0.0f && tau <= 3.402823466e38f;
}
int short_blocks(long long rows, const DeviceCtx* ctx) {
    const long long needed = (rows + kDistilWarps - 1) / kDistilWarps, most = 64LL * ctx->sm_count;
    return static_cast<int>(needed < most ? needed : most);
}

}  // namespace
}  // namespace ldn

using namespace ldn;

extern "C" LDN_API int ldn_distillation(const void* x, long long pitch, long long rows, int V, int type, const void* values, int value_type,
                                        const long long* indices, int k, const long long* targets, float tau, float part, float mix,
                                        float* losses, float* stats, float loss_scale, float* loss, ldn_stream_t stream) {
    if (!distil_fits(rows, V, type, value_type, k, tau)) return kBadArgument;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (rows > 0 && (!x || !values || !indices || !losses)) return kBadArgument;
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    if (rows > 0) {
        DistilArgs a = {};
        a.x = x; a.pitch = pitch; a.rows = rows; a.V = V;
        a.values = values; a.value_type = value_type; a.k = k; a.indices = indices; a.targets = targets;
        a.tau = tau; a.part = part; a.mix = mix;
        a.losses = losses; a.stats = stats;
        r = with_type(type, [&](auto t) {
            using T = decltype(t);
            if (V <= kShort) return launch_after(distil_short_kernel<T>, short_blocks(rows, ctx), kDistilThreads, 0, st, a);
            // as many CTAs per row as it takes to fill the device twice, each with 4096 classes at least
            int ranks = 1;
            while (ranks < kMostRanks && rows * ranks < 2LL * ctx->sm_count && V / (2 * ranks) >= 4096) ranks *= 2;
            return launch_after_in_clusters(distil_long_kernel<T>, ranks, static_cast<unsigned>(rows * ranks), kDistilThreads, 0, st, a);
        });
        if (r != kOk) return r;
    }
    return loss ? launch_after(distil_mean_kernel, 1, kMeanThreads, 0, st, losses, rows, loss_scale, loss) : kOk;
}

extern "C" LDN_API int ldn_distillation_backward(const void* x, long long pitch, long long rows, int V, int type, const void* values,
                                                 int value_type, const long long* indices, int k, const long long* targets, float tau,
                                                 float part, float mix, const float* stats, const float* up, int up_per_row, float up_scale,
                                                 void* grad, ldn_stream_t stream) {
    if (!distil_fits(rows, V, type, value_type, k, tau)) return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !values || !indices || !stats || !up || !grad) return kBadArgument;
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    DistilArgs a = {};
    a.x = x; a.pitch = pitch; a.rows = rows; a.V = V;
    a.values = values; a.value_type = value_type; a.k = k; a.indices = indices; a.targets = targets;
    a.tau = tau; a.part = part; a.mix = mix;
    a.stats = const_cast<float*>(stats);
    a.up = up; a.up_step = up_per_row ? 1 : 0; a.up_scale = up_scale; a.grad = grad;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int entry = sizeof(long long) + sizeof(float);
        if (V <= kShort) {
            constexpr auto kernel = distil_grad_short_kernel<T>;
            static OncePerDevice once;
            const int s = once([] { return allow_smem(kernel, kDistilWarps * (kMostEntries + 1) * (sizeof(long long) + sizeof(float))); });
            if (s != kOk) return s;
            return launch_after(kernel, short_blocks(rows, ctx), kDistilThreads, static_cast<size_t>(kDistilWarps) * (k + 1) * entry, st, a);
        }
        int parts = 1;
        while (parts < 64 && rows * parts < 4LL * ctx->sm_count && V / (2 * parts) >= 2048) parts *= 2;
        return launch_after(distil_grad_long_kernel<T>, dim3(static_cast<unsigned>(rows), parts), kDistilThreads, static_cast<size_t>(k + 1) * entry,
                            st, a);
    });
}
