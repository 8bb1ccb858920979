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
    int items;    // pieces per thread, at most (1, 2, 4 or 8)
    bool group;   // rows share blocks
    bool shift;   // some row starts off a 16-byte boundary, or ends off one
    int rows_per_block() const { return group ? threads / lanes : 1; }
};

inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// false: the row does not fit `most` threads with `items` pieces each (a power of two).  Groups have at least least_lanes threads.
inline bool plan_rows(int C, int piece, bool shift, int items, int most, int least_lanes, RowPlan* p) {
    const long long pieces = shift ? (static_cast<long long>(C) + 2 * piece - 2) / piece : C / piece;
    if (pieces > static_cast<long long>(items) * most) return false;
    p->shift = shift;
    p->items = items;
    p->group = pieces <= 32 * items;
    if (p->group) {
        p->lanes = least_lanes;
        while (p->lanes < 32 && p->lanes * items < pieces) p->lanes *= 2;
        p->threads = kGroupThreads;
        while (p->items > 1 && static_cast<long long>(p->lanes) * (p->items / 2) >= pieces) p->items /= 2;
    } else {
        p->lanes = static_cast<int>((pieces + items - 1) / items + 31) / 32 * 32;
        p->threads = p->lanes;
    }
    return true;
}
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
// Raw elements of a piece (0 outside the row)
template <class T, bool SHIFT>
__device__ __forceinline__ uint4 load_piece(const T* row, int c0, int C) {
    if (!SHIFT || (c0 >= 0 && c0 + kPiece<T> <= C)) {
        if (!SHIFT && c0 >= C) return make_uint4(0u, 0u, 0u, 0u);
        return *reinterpret_cast<const uint4*>(row + c0);
    }
    union { uint4 raw; unsigned short half[8]; unsigned word[4]; } u;
    u.raw = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e)
        if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(C)) {
            if constexpr (sizeof(T) == 4) u.word[e] = reinterpret_cast<const unsigned*>(row)[c0 + e];
            else u.half[e] = reinterpret_cast<const unsigned short*>(row)[c0 + e];
        }
    return u.raw;
}
template <class T>
__device__ __forceinline__ void unpack(uint4 raw, float (&v)[kPiece<T>]) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, __half>) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <class T>
__device__ __forceinline__ uint4 pack(const float (&v)[kPiece<T>]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(v[i]);
        } else if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <class T, bool SHIFT>
__device__ __forceinline__ void store_piece(T* row, int c0, int C, uint4 raw) {
    if (!SHIFT || (c0 >= 0 && c0 + kPiece<T> <= C)) {
        if (!SHIFT && c0 >= C) return;
        *reinterpret_cast<uint4*>(row + c0) = raw;
        return;
    }
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e)
        if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(C)) {
            if constexpr (sizeof(T) == 4) reinterpret_cast<unsigned*>(row)[c0 + e] = w[e];
            else reinterpret_cast<unsigned short*>(row)[c0 + e] = static_cast<unsigned short>(w[e / 2] >> 16 * (e % 2));
        }
}
// Parameters of a piece's columns (`none` outside the row, and where there is no parameter)
template <class T, bool SHIFT>
__device__ __forceinline__ void load_params(const void* p, bool wide, int c0, int C, float none, float (&v)[kPiece<T>]) {
    constexpr int V = kPiece<T>;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
    if (!p) return;
    if (!SHIFT) {
        if (c0 >= C) return;
        if (wide) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + c0 + e);
                v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
            }
        } else {
            unpack<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p) + c0), v);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (static_cast<unsigned>(c0 + e) < static_cast<unsigned>(C)) v[e] = param_at<T>(p, wide, c0 + e);
    }
}
// Whether element e of the piece is in the row
template <bool SHIFT>
__device__ __forceinline__ bool in_row(int c0, int e, int C) {
    return SHIFT ? static_cast<unsigned>(c0 + e) < static_cast<unsigned>(C) : c0 < C;
}

// Sums over the threads that share a row, for all of them: over the lanes of a group by shuffles, over a block with one barrier
// (`slots` alternates between two, so that the next sum does not wait for this one's readers)
struct RowSum {
    int lanes;
    float* slots;  // [2][32][K]
    int turn;
    template <int K, bool GROUP>
    __device__ __forceinline__ void sum(float (&v)[K]) {
        if constexpr (GROUP) {
            for (int d = lanes >> 1; d > 0; d >>= 1)
#pragma unroll
                for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], d);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
            float* s = slots + turn * 64;
            turn ^= 1;
            if ((threadIdx.x & 31) == 0)
#pragma unroll
                for (int k = 0; k < K; ++k) s[(threadIdx.x >> 5) * K + k] = v[k];
            __syncthreads();
            const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = warp_sum(lane < warps ? s[lane * K + k] : 0.0f);
        }
    }
    template <bool GROUP>
    __device__ __forceinline__ unsigned largest(unsigned v) {
        if constexpr (GROUP) {
            for (int d = lanes >> 1; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
        } else {
            v = __reduce_max_sync(0xffffffffu, v);
            unsigned* s = reinterpret_cast<unsigned*>(slots + turn * 64);
            turn ^= 1;
            if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
            __syncthreads();
            const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
            v = __reduce_max_sync(0xffffffffu, lane < warps ? s[lane] : 0u);
        }
        return v;
    }
};
#endif  // __CUDACC__

}  // namespace ldn
