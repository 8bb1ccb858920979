// Distillation from a teacher's top logits, mixed with the cross-entropy of labels, and its gradient:
//     p = softmax(t / tau) over the entries of a row's list,   q = softmax(x / tau) over all classes,
//     loss = part tau^2 sum p (log p - log q) + mix (log sum e^x - x[label]),
//     dx = up (part tau (q - p) + mix (softmax(x) - [label])).
// A list's entry below 0 is absent, a row without entries has no first term, a row with a label below 0 no second; an index beyond the
// classes makes the row's loss and gradient not-a-numbers.
//
// Bound by memory: forward x once (the largest logit and both sums come of one pass, the sums rescaled when a larger logit comes),
// backward x and dx once: the gradient of a row is written whole as if it had no list, and then at the list's classes.
// 8192 x 40001 bf16, 64 entries: forward 150 us, 4.4 TB/s, backward 240, 5.5; 16 x 131072: 12 and 11; 32768 x 1000 bf16, 20 entries: 43 and 51, by each
// row's own way from its loads to its loss.
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
    float* stats;   // [5][rows]: largest logit, 1 / sums at tau and at 1, the list's largest value, 1 / its sum
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
    static __device__ __forceinline__ void unpack(uint4 raw, float2* v) {
        const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
            else if constexpr (std::is_same_v<T, __half>) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            else v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
    }
    // a piece at either end, `none` outside the row
    __device__ __forceinline__ void edge(int j, float none, float2* v) const {
        auto at = [&](int c) { return static_cast<unsigned>(c) < static_cast<unsigned>(V) ? to_float(row[c]) : none; };
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = make_float2(at(first(j) + 2 * i), at(first(j) + 2 * i + 1));
    }
};

// 2 N values, two at a time
// How a row's sums are made: at both temperatures where it has a label and tau is not 1; `squares`: where tau is 2 or 4, e^d is
// e^(d / tau) squared once or twice (32-bit products beside powers of two, of which an SM makes 16 per clock: with a second
// one, 8192 x 40001 bf16 took 215 us, with one 152; a square's error is twice its root's 2^-22, and four times at 4: 1e-6 of a sum whose additions
// round by as much)
struct Way {
    float c, c1;
    bool second;
    int squares;
    __device__ __forceinline__ explicit Way(const DistilArgs& a)
        : c(kLog2e / a.tau), c1(kLog2e), second(a.targets && a.tau != 1.0f), squares(a.tau == 2.0f ? 1 : a.tau == 4.0f ? 2 : 0) {}
};
template <int N>
__device__ __forceinline__ void add_values(Sums& a, const float2 (&v)[N], const Way& way) {
    const float c = way.c, c1 = way.c1;
    float top = largest_of(v[0].x, v[0].y);
#pragma unroll
    for (int i = 1; i < N; ++i) asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(v[i].x), "f"(v[i].y));
    if (!(top <= a.m)) {
        a.s *= exp2_fast((a.m - top) * c);
        a.s1 *= exp2_fast((a.m - top) * c1);
        a.m = top;
    }
    if (a.m == minus_infinity()) return;
    const float2 m = make_float2(-a.m, -a.m), by = make_float2(c, c);
    float2 sum = make_float2(0.0f, 0.0f);
    if (way.second && way.squares) {
        float2 sum1 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 d = __fmul2_rn(__fadd2_rn(v[i], m), by), e = make_float2(exp2_fast(d.x), exp2_fast(d.y));
            float2 q = __fmul2_rn(e, e);
            if (way.squares == 2) q = __fmul2_rn(q, q);
            sum = __fadd2_rn(sum, e);
            sum1 = __fadd2_rn(sum1, q);
        }
        a.s += sum.x + sum.y;
        a.s1 += sum1.x + sum1.y;
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 d = __fmul2_rn(__fadd2_rn(v[i], m), by);
        sum = __fadd2_rn(sum, make_float2(exp2_fast(d.x), exp2_fast(d.y)));
    }
    a.s += sum.x + sum.y;
    if (way.second) {
        const float2 by1 = make_float2(c1, c1);
        sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 d = __fmul2_rn(__fadd2_rn(v[i], m), by1);
            sum = __fadd2_rn(sum, make_float2(exp2_fast(d.x), exp2_fast(d.y)));
        }
        a.s1 += sum.x + sum.y;
    }
}

__device__ __forceinline__ float value_at(const DistilArgs& a, long long i) {
    return a.value_type == LDN_F32 ? static_cast<const float*>(a.values)[i]
         : a.value_type == LDN_F16 ? __half2float(static_cast<const __half*>(a.values)[i])
                                   : __bfloat162float(static_cast<const __nv_bfloat16*>(a.values)[i]);
}

// Sums, and the largest, over the LANES threads that share a row: lanes of a warp (a power of two), or a block with a
// number per warp at `slots`
template <int LANES, class Op>
__device__ __forceinline__ float over_row(float v, Op op, float* slots) {
#pragma unroll
    for (int d = (LANES < 32 ? LANES : 32) / 2; d > 0; d >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, d));
    if constexpr (LANES > 32) {
        if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
        __syncthreads();
        v = slots[0];
#pragma unroll
        for (int w = 1; w < LANES / 32; ++w) v = op(v, slots[w]);
    }
    return v;
}
struct Plus {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Largest {
    __device__ __forceinline__ float operator()(float a, float b) const { return largest_of(a, b); }
};

// What of a row's loss does not wait for its sums: with t = (value - top) / tau (values may be the type's lowest), p = e^t / sum, and the largest of the list's logits as reference,
// terms = sum p (t - log sum - (x - reference) / tau)
struct List {
    float top, inv_sum, terms, reference, target;
    bool some, label, bad;
};
template <class T, int LANES>
__device__ __forceinline__ List read_list(const DistilArgs& a, long long row, float* slots) {
    constexpr int kWarps = LANES > 32 ? LANES / 32 : 0;  // (a block's rounds have slots of their own)
    constexpr int kHeld = LANES > 32 ? 1 : 4;            // a lane's first entries: asked for together, and kept
    const int lane = threadIdx.x & (LANES - 1);
    const T* x = static_cast<const T*>(a.x) + row * a.pitch;
    const long long *indices = a.indices + row * a.k, target = a.targets ? a.targets[row] : -1;
    const float inv_tau = 1.0f / a.tau;
    float bad = target >= a.V ? 1.0f : 0.0f, top = minus_infinity(), reference = minus_infinity();
    bool there[kHeld];
    float v[kHeld], at[kHeld];
    long long index[kHeld];
#pragma unroll
    for (int e = 0; e < kHeld; ++e) {
        const int j = lane + e * LANES;
        index[e] = j < a.k ? indices[j] : -1;
        v[e] = j < a.k ? value_at(a, row * a.k + j) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < kHeld; ++e) {
        there[e] = index[e] >= 0;
        if (index[e] >= a.V) bad = 1.0f;
        at[e] = there[e] && index[e] < a.V ? to_float(x[index[e]]) : minus_infinity();
    }
    List l;
    l.target = target >= 0 && target < a.V ? to_float(x[target]) : 0.0f;
    l.label = target >= 0;
#pragma unroll
    for (int e = 0; e < kHeld; ++e) {
        if (there[e]) top = largest_of(top, v[e]);
        reference = largest_of(reference, at[e]);
    }
    for (int j = lane + kHeld * LANES; j < a.k; j += LANES) {
        const long long i = indices[j];
        if (i >= a.V) bad = 1.0f;
        if (i >= 0) top = largest_of(top, value_at(a, row * a.k + j));
        if (i >= 0 && i < a.V) reference = largest_of(reference, to_float(x[i]));
    }
    l.bad = over_row<LANES>(bad, Largest(), slots) != 0.0f;
    l.top = top = over_row<LANES>(top, Largest(), slots + kWarps);
    l.reference = reference = over_row<LANES>(reference, Largest(), slots + 2 * kWarps);
    l.some = top != minus_infinity();  // (a list of nothing but minus infinity says nothing)
    float sum = 0.0f;
    if (l.some) {
#pragma unroll
        for (int e = 0; e < kHeld; ++e)
            if (there[e]) sum += expf((v[e] - top) * inv_tau);
        for (int j = lane + kHeld * LANES; j < a.k; j += LANES)
            if (indices[j] >= 0) sum += expf((value_at(a, row * a.k + j) - top) * inv_tau);
    }
    sum = over_row<LANES>(sum, Plus(), slots + 3 * kWarps);
    l.inv_sum = 1.0f / sum;
    const float log_sum = logf(sum);
    auto term = [&](float value, float logit) {
        const float t = (value - top) * inv_tau, p = expf(t) * l.inv_sum;
        return p != 0.0f ? p * ((t - log_sum) - (logit - reference) * inv_tau) : 0.0f;
    };
    float terms = 0.0f;
    if (l.some && !l.bad) {
#pragma unroll
        for (int e = 0; e < kHeld; ++e)
            if (there[e]) terms += term(v[e], at[e]);
        for (int j = lane + kHeld * LANES; j < a.k; j += LANES)
            if (indices[j] >= 0) terms += term(value_at(a, row * a.k + j), to_float(x[indices[j]]));
    }
    l.terms = over_row<LANES>(terms, Plus(), slots + 4 * kWarps);
    return l;
}
// The rest, by one lane: the loss, and what the backward pass needs
__device__ __forceinline__ void finish_row(const DistilArgs& a, long long row, const List& l, const Sums& sums) {
    const float s1 = a.tau == 1.0f ? sums.s : sums.s1;
    const bool list = l.some && a.part != 0.0f, label = l.label && a.mix != 0.0f;  // (a term without weight is none, infinite ones too)
    float loss = 0.0f;
    // (a preferred class that is no choice: infinity, whatever the others are)
    if (list) loss = a.part * a.tau * a.tau * (l.reference == minus_infinity() ? -minus_infinity() : l.terms - ((l.reference - sums.m) / a.tau - logf(sums.s)));
    if (label) loss += a.mix * (logf(s1) - (l.target - sums.m));
    a.losses[row] = l.bad ? not_a_number() : loss;
    if (a.stats) {
        a.stats[row] = sums.m;
        a.stats[a.rows + row] = l.bad ? not_a_number() : 1.0f / sums.s;
        a.stats[2 * a.rows + row] = l.bad ? not_a_number() : 1.0f / s1;
        a.stats[3 * a.rows + row] = l.top;
        a.stats[4 * a.rows + row] = l.bad ? not_a_number() : list ? l.inv_sum : 0.0f;
    }
}

// Short rows: some lanes of a warp (distil_lanes).  Longer ones: a block, or the blocks of a cluster, each with a range of the pieces.
constexpr int kAhead = 4;
constexpr int kShortEntries = 128;  // of a list, in the backward pass
// The pieces from `first` to in front of `last`, by a thread of some.  Four are loaded while the four in front of them are worked on (without:
// 8192 x 40001 bf16 178 us); those at a row's cut ends, element by element, come last.
// meanwhile: what is done with the first four under way.
template <class T, class F>
__device__ __forceinline__ void read_pieces(const Pieces<T>& p, int first, int last, int thread, int threads, const Way& way, Sums& sums,
                                            F meanwhile) {
    constexpr int H = Pieces<T>::N / 2;
    if (first >= last) {
        meanwhile();
        return;
    }
    const int begin = p.whole(first) ? first : first + 1, end = p.whole(last - 1) ? last : last - 1;
    int j = begin + thread;
    uint4 raw[kAhead];
    auto load = [&] {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) raw[u] = p.load(j + u * threads);
    };
    bool more = j + (kAhead - 1) * threads < end;
    if (more) load();
    meanwhile();
    while (more) {
        float2 v[kAhead * H];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) Pieces<T>::unpack(raw[u], v + u * H);
        j += kAhead * threads;
        more = j + (kAhead - 1) * threads < end;
        if (more) load();
        add_values(sums, v, way);
    }
    for (; j < end; j += threads) {
        float2 v[H];
        Pieces<T>::unpack(p.load(j), v);
        add_values(sums, v, way);
    }
    if (begin > first && thread == 0) {
        float2 v[H];
        p.edge(first, minus_infinity(), v);
        add_values(sums, v, way);
    }
    if (end < last && last - 1 >= begin && thread == 1) {
        float2 v[H];
        p.edge(last - 1, minus_infinity(), v);
        add_values(sums, v, way);
    }
}

template <class T, int LANES>
__global__ void __launch_bounds__(kDistilThreads, 3) distil_short_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    constexpr int kRows = kDistilThreads / LANES;
    const Way way(a);
    const int lane = threadIdx.x & (LANES - 1);
    for (long long row0 = static_cast<long long>(blockIdx.x) * kRows; row0 < a.rows; row0 += static_cast<long long>(gridDim.x) * kRows) {
        const bool there = row0 + threadIdx.x / LANES < a.rows;  // (lanes without a row of their own go along with the last one)
        const long long row = there ? row0 + threadIdx.x / LANES : a.rows - 1;
        const Pieces<T> p(static_cast<const T*>(a.x) + row * a.pitch, a.V);
        Sums sums = {minus_infinity(), 0.0f, 0.0f};
        List list;
        read_pieces(p, 0, p.count, lane, LANES, way, sums, [&] {
            __syncwarp();
            list = read_list<T, LANES>(a, row, nullptr);
        });
        __syncwarp();
        sums.over_lanes(LANES, way.c, way.c1);
        if (lane == 0 && there) finish_row(a, row, list, sums);
    }
}

// (the first CTA's first warp makes the loss)
template <class T>
__global__ void __launch_bounds__(kDistilThreads, 4) distil_long_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    __shared__ Sums of_warps[kDistilWarps], of_ranks[kMostRanks];
    __shared__ float slots[5 * kDistilWarps];
    __shared__ List list;
    const Way way(a);
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const long long row = blockIdx.x / ranks;
    if (ranks > 1) cluster_barrier();  // (the first CTA is there to be written to)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Pieces<T> p(static_cast<const T*>(a.x) + row * a.pitch, a.V);
    Sums sums = {minus_infinity(), 0.0f, 0.0f};
    read_pieces(p, static_cast<int>(static_cast<long long>(p.count) * rank / ranks), static_cast<int>(static_cast<long long>(p.count) * (rank + 1) / ranks),
                threadIdx.x, kDistilThreads, way, sums, [&] {
                    if (rank != 0) return;
                    const List l = read_list<T, kDistilThreads>(a, row, slots);
                    if (threadIdx.x == 0) list = l;
                });
    __syncwarp();
    sums.over_lanes(32, way.c, way.c1);
    if (lane == 0) of_warps[warp] = sums;
    __syncthreads();
    if (warp == 0) {
        sums = lane < kDistilWarps ? of_warps[lane] : Sums{minus_infinity(), 0.0f, 0.0f};
        sums.over_lanes(kDistilWarps, way.c, way.c1);
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
            sums.over_lanes(kMostRanks, way.c, way.c1);
        }
    }
    if (rank == 0 && threadIdx.x == 0) finish_row(a, row, list, sums);
}

// Many long rows: blocks that take rows in turn and have the next 16 KB pieces of them under way whatever the row that they are of, so that
// nothing waits while a row ends.  A warp fetches, eight add up, one reads the lists and makes the losses.
constexpr int kRingStages = 6, kRingPieces = 1024, kRingBytes = kRingPieces * 16;
constexpr int kRingThreads = kDistilThreads + 64;
constexpr int kRingEntries = 128;  // of a list that one warp reads while a row comes
struct RingBarriers {
    uint64_t full[kRingStages], empty[kRingStages], added[2], taken[2];
};
constexpr int kRingSmem = kRingStages * kRingBytes + 128;
__device__ __forceinline__ void fetch_bytes(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <class T>
__global__ void __launch_bounds__(kRingThreads, 2) distil_ring_kernel(const __grid_constant__ DistilArgs a, int* status) {
    extern __shared__ char raw[];
    char* ring = raw + ((128 - (smem_u32(raw) & 127)) & 127);
    __shared__ RingBarriers B;
    __shared__ Sums of_warps[2][kDistilWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kRingStages; ++s) {
            mbar_init(&B.full[s], 1);
            mbar_init(&B.empty[s], kDistilWarps);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&B.added[s], kDistilWarps);
            mbar_init(&B.taken[s], 1);
        }
        mbar_fence_init();
    }
    __syncthreads();
    stream_order_begin();
    constexpr int H = Pieces<T>::N / 2;
    const Way way(a);
    auto give_up = [&] { atomicExch(status, static_cast<int>(kDeviceTimeout)); };
    // a row's whole pieces (those at its cut ends are the last warp's)
    auto whole_of = [](const Pieces<T>& p, int& begin, int& end) {
        begin = p.whole(0) ? 0 : 1;
        end = p.whole(p.count - 1) ? p.count : p.count - 1;
    };
    auto pieces_of = [&](long long row) { return Pieces<T>(static_cast<const T*>(a.x) + row * a.pitch, a.V); };
    RingPlace<kRingStages> at;
    if (warp == kDistilWarps) {
        if (elected()) {
            long long i = 0;
            bool fine = true;
            for (long long row = blockIdx.x; row < a.rows && fine; row += gridDim.x) {
                const Pieces<T> p = pieces_of(row);
                int j, end;
                whole_of(p, j, end);
                for (; j < end; j += kRingPieces, ++i, at.next()) {
                    if (i >= kRingStages && !mbar_wait_bounded(&B.empty[at.stage], at.parity ^ 1)) {
                        fine = false;
                        give_up();
                        break;
                    }
                    const uint32_t bytes = static_cast<uint32_t>(end - j < kRingPieces ? end - j : kRingPieces) * 16;
                    mbar_expect_tx(&B.full[at.stage], bytes);
                    fetch_bytes(ring + at.stage * kRingBytes, p.row + p.first(j), bytes, &B.full[at.stage]);
                }
            }
            for (long long k = i < kRingStages ? 0 : i - kRingStages; k < i; ++k)  // (no copy is in flight when the block ends)
                if (!mbar_wait_bounded(&B.full[k % kRingStages], (k / kRingStages) & 1)) give_up();
        }
    } else if (warp < kDistilWarps) {
        int n = 0;
        bool fine = true;
        for (long long row = blockIdx.x; row < a.rows && fine; row += gridDim.x, ++n) {
            const Pieces<T> p = pieces_of(row);
            int j, end;
            whole_of(p, j, end);
            Sums sums = {minus_infinity(), 0.0f, 0.0f};
            for (; j < end && fine; j += kRingPieces, at.next()) {
                fine = __all_sync(0xffffffffu, mbar_wait_bounded(&B.full[at.stage], at.parity));
                if (!fine) break;
                const uint4* from = reinterpret_cast<const uint4*>(ring + at.stage * kRingBytes) + threadIdx.x;
                const int left = end - j - static_cast<int>(threadIdx.x);
                static_assert(kRingPieces == kAhead * kDistilThreads, "four pieces per thread");
                if (left > (kAhead - 1) * kDistilThreads) {
                    float2 v[kAhead * H];
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) Pieces<T>::unpack(from[u * kDistilThreads], v + u * H);
                    add_values(sums, v, way);
                } else {
#pragma unroll 1
                    for (int u = 0; u * kDistilThreads < left; ++u) {
                        float2 v[H];
                        Pieces<T>::unpack(from[u * kDistilThreads], v);
                        add_values(sums, v, way);
                    }
                }
                __syncwarp();
                if (lane == 0) arrive(&B.empty[at.stage]);
            }
            sums.over_lanes(32, way.c, way.c1);
            if (n >= 2 && fine) fine = __all_sync(0xffffffffu, mbar_wait_bounded(&B.taken[n & 1], (n / 2 - 1) & 1));
            if (lane == 0 && fine) {
                of_warps[n & 1][warp] = sums;
                arrive(&B.added[n & 1]);
            }
        }
        if (!fine) give_up();
    } else {
        int n = 0;
        for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, ++n) {
            const Pieces<T> p = pieces_of(row);
            // the elements at the row's ends that are in no whole piece
            int begin, end;
            whole_of(p, begin, end);
            const int head = begin ? (p.first(1) < a.V ? p.first(1) : a.V) : 0, tail = end < p.count && end >= begin ? p.first(end) : a.V;
            const int mine = lane < 16 ? lane : tail + lane - 16;
            const bool there = lane < 16 ? mine < head : mine < a.V;
            const float e = there ? to_float(p.row[mine]) : minus_infinity();
            const float one = e == minus_infinity() ? 0.0f : exp2_fast(e - e);  // (not a number for infinity, as in a whole piece)
            Sums sums = {e, one, one};
            const List list = read_list<T, 32>(a, row, nullptr);
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&B.added[n & 1], (n / 2) & 1))) {
                give_up();
                break;
            }
            if (lane < kDistilWarps) {
                const Sums w = of_warps[n & 1][lane];
                sums.join(w.m, w.s, w.s1, way.c, way.c1);
            }
            __syncwarp();
            if (lane == 0) arrive(&B.taken[n & 1]);
            sums.over_lanes(32, way.c, way.c1);
            if (lane == 0) finish_row(a, row, list, sums);
        }
    }
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

// index, minus: room for a list and a label, in whole fours
__host__ __device__ __forceinline__ int list_room(int k) { return (k + 4) / 4 * 4; }
template <class T, int THREADS>
__device__ __forceinline__ void gradient_of_row(const DistilArgs& a, long long row, int part, int parts, int thread, int* index, float* minus, bool there) {
    constexpr int N = Pieces<T>::N;
    const T* x = static_cast<const T*>(a.x) + row * a.pitch;
    T* to = static_cast<T*>(a.grad) + row * a.V;
    const float up = a.up[row * a.up_step] * a.up_scale;
    const float inv_sum = a.stats[4 * a.rows + row], top = a.stats[3 * a.rows + row], inv_tau = 1.0f / a.tau;
    const long long target = a.targets ? a.targets[row] : -1;
    const bool list = inv_sum != 0.0f, label = target >= 0 && a.mix != 0.0f;  // (a list that is not a number is there)
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
    const int first = static_cast<int>(static_cast<long long>(p.count) * part / parts);
    int last_piece = static_cast<int>(static_cast<long long>(p.count) * (part + 1) / parts);
    const int begin = p.first(first) > 0 ? p.first(first) : 0, end = !there ? 0 : p.first(last_piece) < a.V ? p.first(last_piece) : a.V;
    // the list, and the label behind it
    const int room = list_room(a.k);
    for (int j = thread; j < room; j += THREADS) {
        const long long i = j < a.k ? a.indices[row * a.k + j] : j == a.k ? target : -1;
        index[j] = i >= 0 && i < a.V ? static_cast<int>(i) : -1;
        minus[j] = j == a.k ? by_label : j < a.k && i >= 0 && list ? by_list * (expf((value_at(a, row * a.k + j) - top) * inv_tau) * inv_sum) : 0.0f;
    }
    if (!there) last_piece = first;
    const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(to)) & 15u) == 0;
    constexpr int kRow = 2;
    if (same) {
        for (int j0 = first + thread; j0 < last_piece; j0 += kRow * THREADS) {
            uint4 raw[kRow];
#pragma unroll
            for (int u = 0; u < kRow; ++u)
                if (j0 + u * THREADS < last_piece && p.whole(j0 + u * THREADS)) raw[u] = p.load(j0 + u * THREADS);
#pragma unroll
            for (int u = 0; u < kRow; ++u) {
                const int j = j0 + u * THREADS;
                if (j >= last_piece) continue;
                if (p.whole(j)) {
                    float2 v[N / 2];
                    Pieces<T>::unpack(raw[u], v);
                    T e[N];
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        e[2 * i] = from_float<T>(g(v[i].x));
                        e[2 * i + 1] = from_float<T>(g(v[i].y));
                    }
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
    if constexpr (THREADS <= 32) __syncwarp();
    else __syncthreads();
    // the list's classes once more: the first entry of a class writes what all its entries take off
    for (int j = thread; j <= a.k; j += THREADS) {
        const int i = index[j];
        if (i < begin || i >= end) continue;
        float off = 0.0f;
        bool own = true;
        for (int o = 0; o < room; o += 4) {
            const int4 q = *reinterpret_cast<const int4*>(index + o);
            if (q.x != i && q.y != i && q.z != i && q.w != i) continue;
            own = own && !((o < j && q.x == i) || (o + 1 < j && q.y == i) || (o + 2 < j && q.z == i) || (o + 3 < j && q.w == i));
            if (q.x == i) off += minus[o];
            if (q.y == i) off += minus[o + 1];
            if (q.z == i) off += minus[o + 2];
            if (q.w == i) off += minus[o + 3];
        }
        if (own) to[i] = from_float<T>(g(to_float(x[i])) - off);
    }
    if constexpr (THREADS <= 32) __syncwarp();
}

template <class T, int LANES>
__global__ void __launch_bounds__(kDistilThreads) distil_grad_short_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    extern __shared__ int4 list[];  // [row of the block][room], then as many floats
    constexpr int kRows = kDistilThreads / LANES;
    const int mine = threadIdx.x / LANES, room = list_room(a.k);
    int* index = reinterpret_cast<int*>(list);
    float* minus = reinterpret_cast<float*>(index + kRows * room);
    for (long long row0 = static_cast<long long>(blockIdx.x) * kRows; row0 < a.rows; row0 += static_cast<long long>(gridDim.x) * kRows) {
        const bool there = row0 + mine < a.rows;
        gradient_of_row<T, LANES>(a, there ? row0 + mine : a.rows - 1, 0, 1, threadIdx.x & (LANES - 1), index + mine * room, minus + mine * room, there);
    }
}
template <class T>
__global__ void __launch_bounds__(kDistilThreads) distil_grad_long_kernel(const __grid_constant__ DistilArgs a) {
    stream_order_begin();
    extern __shared__ int4 list[];
    const int parts = gridDim.y;
    int* index = reinterpret_cast<int*>(list);
    gradient_of_row<T, kDistilThreads>(a, blockIdx.x, blockIdx.y, parts, threadIdx.x, index, reinterpret_cast<float*>(index + list_room(a.k)), true);
}

bool distil_fits(long long rows, int V, int type, int value_type, int k, float tau) {
    return rows >= 0 && rows <= kMostColumns && row_fits(V) && known_type(type) && known_type(value_type) && k >= 1 && k <= kMostEntries &&
           tau > 0.0f && tau <= 3.402823466e38f;
}
// Lanes of a warp that share a row, 0: a block or more per row.  What bounds short rows is the way from a row's loads to its loss, so there are as
// many at once as can be.
int distil_lanes(long long rows, int V, const DeviceCtx* ctx) {
    if (V <= 256) return 8;
    if (V <= 1024) return 16;
    return V <= 2048 || (V <= 8192 && rows >= 16LL * ctx->sm_count) ? 32 : 0;
}
template <class F>
int with_lanes(int lanes, F f) {
    using std::integral_constant;
    return lanes == 8 ? f(integral_constant<int, 8>()) : lanes == 16 ? f(integral_constant<int, 16>()) : f(integral_constant<int, 32>());
}
int short_blocks(long long rows, int lanes, const DeviceCtx* ctx) {
    const int of_block = kDistilThreads / lanes;
    const long long needed = (rows + of_block - 1) / of_block, most = 64LL * ctx->sm_count;
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
            if (const int lanes = distil_lanes(rows, V, ctx))
                return with_lanes(lanes, [&](auto n) {
                    return launch_after(distil_short_kernel<T, decltype(n)::value>, short_blocks(rows, lanes, ctx), kDistilThreads, 0, st, a);
                });
            if (rows >= 4LL * ctx->sm_count && k <= kRingEntries) {
                constexpr auto kernel = distil_ring_kernel<T>;
                static OncePerDevice once;
                int s = once([] { return allow_smem(kernel, kRingSmem); });
                Scratch scratch;  // (for the status word)
                if (s == kOk) s = scratch.take(st, 0);
                if (s != kOk) return s;
                return launch_after(kernel, static_cast<unsigned>(2 * ctx->sm_count), kRingThreads, kRingSmem, st, a, scratch.status);
            }
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
        const size_t of_row = static_cast<size_t>(list_room(k)) * 8;
        const int lanes = k <= kShortEntries ? distil_lanes(rows, V, ctx) : 0;
        if (lanes)
            return with_lanes(lanes, [&](auto n) {
                return launch_after(distil_grad_short_kernel<T, decltype(n)::value>, short_blocks(rows, lanes, ctx), kDistilThreads,
                                    kDistilThreads / lanes * of_row, st, a);
            });
        int parts = 1;
        while (parts < 64 && rows * parts < 4LL * ctx->sm_count && V / (2 * parts) >= 2048) parts *= 2;
        return launch_after(distil_grad_long_kernel<T>, dim3(static_cast<unsigned>(rows), parts), kDistilThreads, of_row, st, a);
    });
}
