// Dropout with a counter-based generator: out = [residual +] (x / (1 - p) where its word says so, else 0).  No mask is stored;
// the backward pass is the same kernel on the gradient with the same seed and offset.
//
// Bound by the latency of the generator's ten dependent rounds in 16 bits (the integer pipe is 58 % busy; its words alone take 50 of
// the 90 us of 16384 x 5120, memory 51), by memory in 32: 50000 x 5120 bf16 takes 258 us (4.0 TB/s), with a residual 304 (5.1);
// 8192 x 5120 f32 61 us (5.5 TB/s).  Any other pitch or alignment: 16384 x 5120 bf16 with a pitch of 5121 170 us.
#include "ldn_rows.cuh"

namespace ldn {
namespace {

struct DropoutCall {
    const void *x, *residual;
    long long pitch, pitch_residual, rows;
    int C;
    DropoutArgs drop;
    void* out;
};

// Contiguous tensors that start at multiples of 16 bytes: 16-byte pieces, the next one under way while a thread has this one's words
// made.
template <class T, bool ONTO>
__global__ void __launch_bounds__(kThreads) dropout_pieces_kernel(DropoutCall a, long long n) {
    stream_order_begin();
    constexpr int V = kPiece<T>;
    const Generator gen = generator_of(a.drop);
    const T *x = static_cast<const T*>(a.x), *onto = static_cast<const T*>(a.residual);
    T* out = static_cast<T*>(a.out);
    const long long pieces = n / V, step = static_cast<long long>(gridDim.x) * kThreads;
    long long piece = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    uint4 next = make_uint4(0u, 0u, 0u, 0u), next_onto = next;
    auto fetch = [&](long long i) {
        if (i < pieces) {
            next = *reinterpret_cast<const uint4*>(x + i * V);
            if (ONTO) next_onto = *reinterpret_cast<const uint4*>(onto + i * V);
        }
    };
    fetch(piece);
    for (; piece < pieces; piece += step) {
        const uint4 raw = next, raw_onto = next_onto;
        fetch(piece + step);
        float2 v[V / 2], r[V / 2];
        unpack<T>(raw, v);
        if (ONTO) unpack<T>(raw_onto, r);
        drop_piece(a.drop, gen, piece * V, v);
        if (ONTO)
#pragma unroll
            for (int e = 0; e < V / 2; ++e) v[e] = __fadd2_rn(r[e], v[e]);
        *reinterpret_cast<uint4*>(out + piece * V) = pack<T>(v);
    }
    // what is left behind the last whole piece
    const long long i = pieces * V + threadIdx.x;
    if (blockIdx.x == 0 && i < n) {
        float v = dropped(a.drop, random_word(gen, i), to_float(x[i]));
        if (ONTO) v = __fadd_rn(to_float(onto[i]), v);
        out[i] = from_float<T>(v);
    }
}

// Any pitch and alignment: a thread has the four elements of a block of words, wherever the rows break.
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
        const long long n = rows * C;
        if (pitch == C && (!residual || pitch_residual == C) && on16(x) && on16(residual) && on16(out)) {
            const long long blocks = (n / kPiece<T> + kThreads - 1) / kThreads + (n < kPiece<T>), most = 6LL * ctx->sm_count;
            const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
            const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
            return residual ? launch_after(dropout_pieces_kernel<T, true>, grid, kThreads, 0, st, a, n)
                            : launch_after(dropout_pieces_kernel<T, false>, grid, kThreads, 0, st, a, n);
        }
        const long long blocks = ((rows * C + 3) / 4 + kThreads - 1) / kThreads, most = 32LL * ctx->sm_count;
        return launch_after(dropout_kernel<T>, static_cast<unsigned>(blocks < most ? blocks : most), kThreads, 0,
                            reinterpret_cast<cudaStream_t>(stream), a);
    });
}
