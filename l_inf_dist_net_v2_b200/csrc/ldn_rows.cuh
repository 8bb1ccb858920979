// Rows held in registers: how a kernel that reads a row once, reduces over it and writes it deals its elements out.
//
// A row is cut at the 16-byte boundaries of memory, so every piece but the first and the last of a row is one aligned load whatever
// the row's length is, and pieces of neighbouring tensors with the same place in their 16 bytes match.  Piece j of a row holds the
// columns j kPiece - shift .. + kPiece - 1, shift being the place of the row's first element.  Thread l of the `lanes` that share a
// row has the pieces l, l + lanes, ...: up to 32 lanes of a warp (several rows per warp then), or a block of whole warps.
#pragma once
#include "ldn_head.cuh"

namespace ldn {

constexpr int kGroupThreads = 256;  // of blocks whose warps have rows of their own

template <class T>
constexpr int kPiece = 16 / sizeof(T);

struct RowPlan {
    int lanes;    // threads per row
    int threads;  // per block
    int items;    // pieces per thread, at most
    bool group;   // rows share blocks
    bool shift;   // some row starts off a 16-byte boundary, or ends off one
    int rows_per_block() const { return group ? threads / lanes : 1; }
};

inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// false: the row does not fit `most` threads with `items` pieces each
inline bool plan_rows(int C, int piece, bool shift, int items, int most, RowPlan* p) {
    const long long pieces = shift ? (static_cast<long long>(C) + 2 * piece - 2) / piece : C / piece;
    if (pieces > static_cast<long long>(items) * most) return false;
    p->shift = shift;
    p->items = items;
    p->group = pieces <= 32 * items;
    if (p->group) {
        p->lanes = 1;
        while (p->lanes < 32 && p->lanes * items < pieces) p->lanes *= 2;
        p->threads = kGroupThreads;
    } else {
        p->lanes = static_cast<int>((pieces + items - 1) / items + 31) / 32 * 32;
        p->threads = p->lanes;
    }
    return true;
}
// Elements per thread.  Rows that share blocks: 16, or 8 where the group is no smaller for it.  Rows with blocks of their own: 16 of 16
// bits, 8 of 32 bits and with the words of a dropout (`heavy`), as that many fill the registers of two blocks of 320 threads or
// one of 640 (8192 x 5120 in 32 bits, us, 8 / 16: norm 59 / 66, gradient 93 / 115, joined 117 / 192 and 161 / 250; 16384 x 5120
// in bf16: 82 / 64, 126 / 115, joined gradient 241 / 293); rows that do not fit them take 32.
constexpr int kThreads8 = 640, kThreads16 = 320, kThreads32 = 512;
inline bool plan_elements(int C, int size, bool shift, bool heavy, RowPlan* p) {
    const int piece = 16 / size;
    if (plan_rows(C, piece, shift, 16 / piece, 32, p)) {
        RowPlan fewer;
        if (plan_rows(C, piece, shift, 8 / piece, 32, &fewer) && fewer.lanes == p->lanes) *p = fewer;
        return true;
    }
    const bool eight = heavy || size == 4;
    if (!plan_rows(C, piece, shift, (eight ? 8 : 16) / piece, eight ? kThreads8 : kThreads16, p) &&
        !plan_rows(C, piece, shift, 32 / piece, kThreads32, p))
        return false;
    return !p->group;
}
__host__ __device__ constexpr int threads_of(int elements) { return elements <= 8 ? kThreads8 : elements <= 16 ? kThreads16 : kThreads32; }
// Rows of contiguous tensors, and of one with a pitch of its own, that can be cut alike
inline bool rows_match(int size, long long C, long long pitch, bool all_on16) {
    return all_on16 && (pitch == C || (pitch * size % 16 == 0 && C * size % 16 == 0));
}
inline bool rows_shift(int size, long long C) { return C * size % 16 != 0; }

#ifdef __CUDACC__
// The place of a row's first element in its 16 bytes
template <class T>
__device__ __forceinline__ int shift_of(const T* row) {
    return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
}
// A row's pieces on their way into shared memory: every thread copies its own and reads them back itself, so nothing waits for
// another thread.  What is behind the row's end is not read (zeros come for it, and slots of pieces behind it are zeros from the
// start); what is in front of the row's start is the end of the row before, and reads as it is, but in front of the tensor, where a
// piece comes element by element.
template <class T>
__device__ __forceinline__ int piece_bytes(int c0, int C) {
    const int left = (C - c0) * static_cast<int>(sizeof(T));
    return left < 0 ? 0 : left < 16 ? left : 16;
}
// from: the place of the piece's first element, of column c0; base: the tensor
template <class T, bool SHIFT>
__device__ __forceinline__ void copy_piece(uint4* slot, const T* from, int c0, int bytes, const void* base) {
    if (SHIFT && c0 < 0 && reinterpret_cast<uintptr_t>(from) < reinterpret_cast<uintptr_t>(base)) {
        alignas(16) T v[kPiece<T>];
#pragma unroll
        for (int e = 0; e < kPiece<T>; ++e) v[e] = c0 + e >= 0 && e * static_cast<int>(sizeof(T)) < bytes ? from[e] : from_float<T>(0.0f);
        *slot = *reinterpret_cast<const uint4*>(v);
    } else if (bytes) {
        copy_async<16>(slot, from, SHIFT ? bytes : 16);
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest n - 1 groups have arrived
__device__ __forceinline__ void copies_wait(int n) {
    if (n >= 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (n == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (n == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
// (in pairs, for the packed arithmetic: half the instructions at the same rate per element)
template <class T>
__device__ __forceinline__ void unpack(uint4 raw, float2 (&v)[kPiece<T> / 2]) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < kPiece<T> / 2; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else if constexpr (std::is_same_v<T, __half>) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
}
template <class T>
__device__ __forceinline__ uint4 pack(const float2 (&v)[kPiece<T> / 2]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < kPiece<T> / 2; ++i) {
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(v[i].x);
            w[2 * i + 1] = __float_as_uint(v[i].y);
        } else if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = __floats2half2_rn(v[i].x, v[i].y);
            w[i] = *reinterpret_cast<const unsigned*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
            w[i] = *reinterpret_cast<const unsigned*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// Bits of the elements of a piece that are in the row; where pieces are not cut, all are (a piece behind the row's end is zeros anyway)
template <class T, bool SHIFT>
__device__ __forceinline__ uint4 mask_of(int c0, int C) {
    unsigned w[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
    if (SHIFT)
#pragma unroll
        for (int e = 0; e < kPiece<T>; ++e)
            if (static_cast<unsigned>(c0 + e) >= static_cast<unsigned>(C)) {
                if constexpr (sizeof(T) == 4) w[e] = 0u;
                else w[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
            }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 masked(uint4 v, uint4 m) { return make_uint4(v.x & m.x, v.y & m.y, v.z & m.z, v.w & m.w); }
template <class T, bool SHIFT>
__device__ __forceinline__ void store_piece(T* to, int c0, int C, uint4 raw) {
    if (!SHIFT || (c0 >= 0 && c0 + kPiece<T> <= C)) {
        if (SHIFT || c0 < C) *reinterpret_cast<uint4*>(to) = raw;
        return;
    }
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e)
        if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(C)) {
            if constexpr (sizeof(T) == 4) reinterpret_cast<unsigned*>(to)[e] = w[e];
            else reinterpret_cast<unsigned short*>(to)[e] = static_cast<unsigned short>(w[e / 2] >> 16 * (e % 2));
        }
}
// Places of a thread's first piece in the rows that it has in turn
template <class T>
struct Walk {
    T* at;
    long long step;
    __device__ __forceinline__ Walk(const void* base, long long pitch, long long row, long long step_rows, int c0)
        : at(static_cast<T*>(const_cast<void*>(base)) + row * pitch + c0), step(step_rows * pitch) {}
    __device__ __forceinline__ T* of(int j, int offset) const { return at + j * step + offset; }
    __device__ __forceinline__ void on(int rows) { at += rows * step; }
};
// Parameters of a piece's columns (`none` outside the row, and where there is no parameter)
template <class T, bool SHIFT>
__device__ __forceinline__ void load_params(const void* p, bool wide, int c0, int C, float none, float2 (&v)[kPiece<T> / 2]) {
    constexpr int V = kPiece<T>;
#pragma unroll
    for (int e = 0; e < V / 2; ++e) v[e] = both(none);
    if (!p) return;
    if (!SHIFT) {
        if (c0 >= C) return;
        if (wide) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + c0 + e);
                v[e / 2] = make_float2(f.x, f.y);
                v[e / 2 + 1] = make_float2(f.z, f.w);
            }
        } else {
            unpack<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p) + c0), v);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(C)) {
                const float f = param_at<T>(p, wide, c0 + e);
                if (e % 2) v[e / 2].y = f;
                else v[e / 2].x = f;
            }
    }
}
// Zeros for the elements outside the row (there are some at its ends only; pieces that are not cut are whole or not there)
template <bool SHIFT, int N>
__device__ __forceinline__ void only_row(int c0, int C, float2 (&v)[N]) {
    if (SHIFT ? c0 < 0 || c0 + 2 * N > C : c0 >= C)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (static_cast<unsigned>(c0 + 2 * e) >= static_cast<unsigned>(C)) v[e].x = 0.0f;
            if (static_cast<unsigned>(c0 + 2 * e + 1) >= static_cast<unsigned>(C)) v[e].y = 0.0f;
        }
}
// Rows of T elements that are under way at a time, if a block may have `budget` bytes for them
inline int ring_depth(long long row_bytes, long long budget) {
    const long long d = budget / row_bytes;
    return d >= 4 ? 4 : static_cast<int>(d);
}

// Sums and maxima over the threads that share a row, for all of them: over the lanes of a group by shuffles, over a block with one
// barrier (`slots` alternates between two, so that the next one does not wait for this one's readers).  A block has K numbers at a
// time, of several rows: the first steps of a warp's tree halve what a lane has to carry, so eight sums take 19 shuffles instead
// of 80.
struct RowSum {
    int lanes;
    float* slots;  // [2][kSlots]
    int turn;
    static constexpr int kSlots = 20 * 8;  // (warps of a block) x K
    template <int K, class Op, class End>
    __device__ __forceinline__ void over_block(float (&v)[K], Op op, End end) {
        const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        constexpr int kShare = 32 / K;  // lanes that end with the same number
        int half = 16;
#pragma unroll
        for (int n = K; n > 1; n /= 2, half /= 2) {
            const bool upper = lane & half;
#pragma unroll
            for (int i = 0; i < n / 2; ++i) {
                const float send = upper ? v[i] : v[i + n / 2], keep = upper ? v[i + n / 2] : v[i];
                v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, half));
            }
        }
#pragma unroll
        for (int d = kShare / 2; d > 0; d /= 2) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], d));
        float* s = slots + turn * kSlots;
        turn ^= 1;
        const int k = lane / kShare, first = lane % kShare;
        if (first == 0) s[(threadIdx.x >> 5) * K + k] = v[0];
        __syncthreads();
        float r = 0.0f;  // (nothing is below it that is not summed: maxima are of magnitudes)
        for (int w = first; w < warps; w += kShare) r = op(r, s[w * K + k]);
#pragma unroll
        for (int d = kShare / 2; d > 0; d /= 2) r = op(r, __shfl_xor_sync(0xffffffffu, r, d));
        r = end(r);
#pragma unroll
        for (int i = 0; i < K; ++i) v[i] = K == 1 ? r : __shfl_sync(0xffffffffu, r, i * kShare);
    }
    template <int K, class Op, class End>
    __device__ __forceinline__ void over_group(float (&v)[K], Op op, End end) {
        for (int d = lanes >> 1; d > 0; d >>= 1)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = op(v[k], __shfl_xor_sync(0xffffffffu, v[k], d));
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = end(v[k]);
    }
    // (what comes of a sum is made of it before it is handed out)
    template <bool GROUP, int K, class End>
    __device__ __forceinline__ void sum(float (&v)[K], End end) {
        auto op = [](float a, float b) { return a + b; };
        if constexpr (GROUP) over_group(v, op, end);
        else over_block(v, op, end);
    }
    template <bool GROUP, int K, class End>
    __device__ __forceinline__ void largest(float (&v)[K], End end) {
        auto op = [](float a, float b) { return larger(a, b); };
        if constexpr (GROUP) over_group(v, op, end);
        else over_block(v, op, end);
    }
};
#endif  // __CUDACC__

}  // namespace ldn
