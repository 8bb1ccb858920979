// The gated projection, forward and backward: operands as the tensor cores' loads want them, the gradients of the two projections, and
// the entry points.
//
// The backward pass needs both projections again.  They are kept in 32 bits: rounded to bfloat16 they took the weights' gradients from
// 2.4e-3 to 3.1e-3 of 64 bits (1.7e-3 is their own rounding), and making them again would cost a third of a training step's products.
// What enters the products as dg and du has the rows' type: the tensor cores multiply no other at that rate, and two numbers of 16 bits for each
// would double the backward pass's products (16384, 5120 -> 5120 bf16: 2.2 ms of 4.4).  For it all three gradients are 2.3e-3 of 64 bits,
// 1.7e-3 of which their own rounding is; in float16 what is below 6e-8 of them is lost, as anywhere in that type.  Bound by memory: dy, both
// projections, both gradients once (16384 x 5120 bf16: 226 us, 5.2 TB/s; 512 x 2048 float32: 9).
#include "ldn_gated.cuh"
#include "ldn_words.cuh"

namespace ldn {
namespace {

long long padded8(long long n) { return (n + 7) / 8 * 8; }
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- operands -----------------------------------------------------------------------------------------------------------------------
struct Source {
    const void* from;
    long long pitch, rows;
    int C;
    unsigned short* to;
    long long pitch_to, apart;
};
struct Sources {
    Source of[3];
};
constexpr int kCopyThreads = 256;

// A number of 32 bits as the sum of three of bfloat16: what each leaves is exact, and 24 bits are all (numbers below 2^-110 lose their
// last bits).  What is not finite is in the first image alone.
__device__ __forceinline__ void split3(float v, unsigned short (&part)[3]) {
    __nv_bfloat16 h = __float2bfloat16_rn(v);
    if (magnitude(v) < 0x7f800000u && magnitude(__bfloat162float(h)) == 0x7f800000u) h = __float2bfloat16_rz(v);
    const bool finite = magnitude(v) < 0x7f800000u;
    const float r1 = finite ? v - __bfloat162float(h) : 0.0f;
    const __nv_bfloat16 m = __float2bfloat16_rn(r1);
    const __nv_bfloat16 l = __float2bfloat16_rn(r1 - __bfloat162float(m));
    part[0] = __bfloat16_as_ushort(h);
    part[1] = __bfloat16_as_ushort(m);
    part[2] = __bfloat16_as_ushort(l);
}
__device__ __forceinline__ uint4 packed8(const unsigned short (&v)[8]) {
    uint4 r;
    r.x = v[0] | static_cast<unsigned>(v[1]) << 16;
    r.y = v[2] | static_cast<unsigned>(v[3]) << 16;
    r.z = v[4] | static_cast<unsigned>(v[5]) << 16;
    r.w = v[6] | static_cast<unsigned>(v[7]) << 16;
    return r;
}
__device__ __forceinline__ void store_split8(unsigned short* to, long long apart, const float (&v)[8]) {
    unsigned short image[3][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        unsigned short part[3];
        split3(v[j], part);
#pragma unroll
        for (int i = 0; i < 3; ++i) image[i][j] = part[i];
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(to + i * apart) = packed8(image[i]);
}
// Rows of any pitch and alignment as images: of 16 bits a copy, of 32 three parts.  A thread has eight columns.  Bound by memory: x and both
// weights of 512, 5120 -> 2048 in float32, 94 MB in and 141 out, 34 us, 6.9 TB/s.
template <class T>
__global__ void __launch_bounds__(kCopyThreads) images_kernel(const __grid_constant__ Sources sources) {
    stream_order_begin();
    const Source& s = sources.of[blockIdx.y];
    const unsigned pieces = static_cast<unsigned>(s.pitch_to / 8);
    const long long all = s.rows * pieces, step = static_cast<long long>(gridDim.x) * kCopyThreads;
    const bool whole = sizeof(T) == 4 && ((reinterpret_cast<uintptr_t>(s.from) | (s.pitch * sizeof(T))) & 15u) == 0;
    for (long long i = static_cast<long long>(blockIdx.x) * kCopyThreads + threadIdx.x; i < all; i += step) {
        const long long row = (all >> 32) == 0 ? static_cast<unsigned>(i) / pieces : i / pieces;
        const int c = static_cast<int>(i - row * pieces) * 8;
        const T* from = static_cast<const T*>(s.from) + row * s.pitch + c;
        unsigned short* to = s.to + row * s.pitch_to + c;
        if constexpr (sizeof(T) == 4) {
            float v[8];
            if (whole && c + 8 <= s.C) {
                const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = c + j < s.C ? from[j] : 0.0f;
            }
            store_split8(to, s.apart, v);
        } else {
            // a piece that starts anywhere, from the two words of memory that it lies in, where both are the tensor's
            const unsigned off = static_cast<unsigned>(reinterpret_cast<uintptr_t>(from) & 15u);
            const int words = words_of_piece(off, c, s.C, row, s.rows, s.pitch);
            if (words == 1) {
                *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
            } else if (words == 2) {
                const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(from) - off);
                const uint4 a = at[0], b = at[1];
                const unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                const unsigned first = off / 4, bits = off % 4 * 8;
                auto word = [&](unsigned i) { return i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : i == 3 ? w[3] : i == 4 ? w[4] : i == 5 ? w[5] : i == 6 ? w[6] : w[7]; };
                unsigned v[5];
#pragma unroll
                for (unsigned i = 0; i < 5; ++i) v[i] = word(first + i);
                *reinterpret_cast<uint4*>(to) = make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits),
                                                           __funnelshift_r(v[2], v[3], bits), __funnelshift_r(v[3], v[4], bits));
            } else {
                unsigned short v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = c + j < s.C ? reinterpret_cast<const unsigned short*>(from)[j] : 0;
                *reinterpret_cast<uint4*>(to) = packed8(v);
            }
        }
    }
}

// Operands on their way into images: which are read where they lie, and what the others take of scratch
struct Operands {
    int type;
    Sources sources = {};
    Images images[3];
    int count = 0, copies = 0;
    int copied[3];
    size_t bytes = 0;

    // the operand's number
    int add(const void* p, long long pitch, long long rows, int C) {
        Images& o = images[count];
        o.rows = rows;
        o.columns = C;
        if (type != LDN_F32 && on16(p) && ((pitch >= C && pitch % 8 == 0) || rows == 1)) {
            o.base = p;
            o.pitch = rows == 1 ? padded8(C) : pitch;
        } else {
            o.pitch = padded8(C);
            o.apart = rows * o.pitch;
            o.count = type == LDN_F32 ? 3 : 1;
            copied[copies] = count;
            sources.of[copies++] = {p, pitch, rows, C, nullptr, o.pitch, o.apart};
            bytes += pad256(static_cast<size_t>(o.count) * o.apart * 2);
        }
        return count++;
    }
    // (in images that are there already)
    void found(char* at) {
        for (int i = 0; i < copies; ++i) {
            Images& o = images[copied[i]];
            o.base = at;
            at += pad256(static_cast<size_t>(o.count) * o.apart * 2);
        }
        copies = 0;
        bytes = 0;
    }
    int launch(char* scratch, const DeviceCtx* ctx, cudaStream_t st) {
        if (!copies) return kOk;
        long long most = 0;
        for (int i = 0; i < copies; ++i) {
            Images& o = images[copied[i]];
            o.base = scratch;
            sources.of[i].to = reinterpret_cast<unsigned short*>(scratch);
            scratch += pad256(static_cast<size_t>(o.count) * o.apart * 2);
            const long long items = o.rows * (o.pitch / 8);
            if (items > most) most = items;
        }
        const long long blocks = (most + kCopyThreads - 1) / kCopyThreads, cap = 16LL * ctx->sm_count;
        const dim3 grid(static_cast<unsigned>(blocks < cap ? blocks : cap), copies);
        return with_type(type, [&](auto t) { return launch_after(images_kernel<decltype(t)>, grid, kCopyThreads, 0, st, sources); });
    }
};

// ---- gradients of the projections --------------------------------------------------------------------------------------------------
struct GradArgs {
    const void* grad_y;  // [T][H]
    const float *g, *u;  // [T][pitch_saved]
    long long pitch_saved, T;
    int H;
    unsigned short* to;  // [side][part][T][pitch_to]
    long long pitch_to, apart;
    float* sums;  // [block of rows][2][H], may be null
};
constexpr int kGradLanes = 32, kGradRows = 8, kGradColumns = kGradLanes * 8;

template <class T>
__device__ __forceinline__ void load8(const T* p, bool whole, int there, float (&v)[8]) {
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

// Eight kept numbers at a multiple of 32 bytes
__device__ __forceinline__ void load_kept(const float* p, int there, float (&v)[8]) {
    if (there >= 8) {
        asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "l"(p));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < there ? p[j] : 0.0f;
    }
}

// dg = dy u act'(g), du = dy act(g) as images, and their column sums over a block of rows: a thread has eight columns and every eighth row.
// (Told its activation when it is compiled: asked for at each element, 16384 x 5120 bf16 took 253 us.)
template <class T, int ACTIVATION>
__global__ void __launch_bounds__(kGradLanes * kGradRows, 4) gated_grad_kernel(const __grid_constant__ GradArgs a) {
    stream_order_begin();
    __shared__ float sums[kGradRows][2][kGradColumns];
    const int lane = threadIdx.x % kGradLanes, part = threadIdx.x / kGradLanes, c = blockIdx.x * kGradColumns + lane * 8, there = a.H - c;
    const bool whole = ((reinterpret_cast<uintptr_t>(a.grad_y) | (static_cast<size_t>(a.H) * sizeof(T))) & 15u) == 0 && there >= 8;
    constexpr int kImages = sizeof(T) == 4 ? 3 : 1;
    float sg[8] = {}, su[8] = {};
    const long long step = static_cast<long long>(gridDim.y) * kGradRows;
    if (there > 0)
        for (long long row = static_cast<long long>(blockIdx.y) * kGradRows + part; row < a.T; row += step) {
            float dy[8], g[8], u[8], dg[8], du[8];
            load8(static_cast<const T*>(a.grad_y) + row * a.H + c, whole, there, dy);
            load_kept(a.g + row * a.pitch_saved + c, there, g);
            load_kept(a.u + row * a.pitch_saved + c, there, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 f = activation_and_slope(g[j], ACTIVATION);
                dg[j] = dy[j] * u[j] * f.y;
                du[j] = dy[j] * f.x;
                sg[j] += dg[j];
                su[j] += du[j];
            }
            unsigned short* to = a.to + row * a.pitch_to + c;
            if constexpr (kImages == 3) {
                store_split8(to, a.apart, dg);
                store_split8(to + 3 * a.apart, a.apart, du);
            } else {
                unsigned short v[2][8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const T p = from_float<T>(dg[j]), q = from_float<T>(du[j]);
                    v[0][j] = *reinterpret_cast<const unsigned short*>(&p);
                    v[1][j] = *reinterpret_cast<const unsigned short*>(&q);
                }
                *reinterpret_cast<uint4*>(to) = packed8(v[0]);
                *reinterpret_cast<uint4*>(to + a.apart) = packed8(v[1]);
            }
        }
    if (!a.sums) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        sums[part][0][lane * 8 + j] = sg[j];
        sums[part][1][lane * 8 + j] = su[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * kGradColumns; i += kGradLanes * kGradRows) {
        const int side = i / kGradColumns, column = i % kGradColumns, n = blockIdx.x * kGradColumns + column;
        if (n >= a.H) continue;
        float s = 0.0f;
#pragma unroll
        for (int r = 0; r < kGradRows; ++r) s += sums[r][side][column];
        a.sums[(static_cast<long long>(blockIdx.y) * 2 + side) * a.H + n] = s;
    }
}

// The blocks' sums in order: a thread has a column of one of the two and every eighth part.
constexpr int kFoldColumns = 32, kFoldLanes = 8;
template <class T>
__global__ void __launch_bounds__(kFoldColumns * kFoldLanes) gated_fold_kernel(const float* parts, int count, int H, bool wide, void* grad_gate,
                                                                              void* grad_up) {
    stream_order_begin();
    __shared__ float sums[kFoldLanes][kFoldColumns];
    const int lane = threadIdx.x % kFoldColumns, part = threadIdx.x / kFoldColumns, c = blockIdx.x * kFoldColumns + lane;
    float s = 0.0f;
    if (c < H)
        for (int i = part; i < count; i += kFoldLanes) s += parts[(2LL * i + blockIdx.y) * H + c];
    sums[part][lane] = s;
    __syncthreads();
    void* to = blockIdx.y ? grad_up : grad_gate;
    if (part == 0 && c < H && to) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < kFoldLanes; ++i) s += sums[i][lane];
        set_param<T>(to, wide, c, s);
    }
}

bool gated_fits(long long T, int K, int H, int type, int param_type, const void* b_gate, const void* b_up, int activation,
                long long pitch_gate, long long pitch_up) {
    return T >= 0 && T <= kMostColumns && row_fits(K) && row_fits(H) && known_type(type) && gated_activation(activation) &&
           pitch_gate >= K && pitch_up >= K && ((!b_gate && !b_up) || param_type == LDN_F32 || param_type == type);
}
bool on32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }

}  // namespace
}  // namespace ldn

using namespace ldn;

extern "C" LDN_API unsigned long long ldn_gated_image_bytes(long long rows, int K, int H, int type) {
    GatedArgs a = {};
    a.T = rows;
    if (type != LDN_F32 || rows < 1 || !row_fits(K) || !row_fits(H) || gated_is_few(a, type)) return 0;
    Operands o{type};
    for (const long long n : {rows, static_cast<long long>(H), static_cast<long long>(H)}) o.add(nullptr, K, n, K);
    return o.bytes;
}

extern "C" LDN_API int ldn_gated_linear(const void* x, long long pitch, long long rows, int K, int H, int type, const void* w_gate,
                                        long long pitch_gate, const void* w_up, long long pitch_up, const void* b_gate, const void* b_up,
                                        int param_type, int activation, void* y, float* g, float* u, long long pitch_saved,
                                        void* images, ldn_stream_t stream) {
    if (!gated_fits(rows, K, H, type, param_type, b_gate, b_up, activation, pitch_gate, pitch_up) || !g != !u) return kBadArgument;
    if (g && (pitch_saved < H || pitch_saved % 16 || !on32(g) || !on32(u))) return kBadArgument;
    if (rows == 0) return kOk;
    if (!x || !w_gate || !w_up || !y) return kBadArgument;
    const DeviceCtx* ctx;
    int r = get_device_ctx(&ctx);
    if (r != kOk) return r;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const GatedArgs a = {x, pitch, w_gate, w_up, pitch_gate, pitch_up, b_gate, b_up, param_type == LDN_F32, rows, K, H, activation, y, g, u,
                         pitch_saved};
    if (gated_is_few(a, type)) return launch_gated_few(a, type, st);
    Operands o{type};
    o.add(x, pitch, rows, K);
    o.add(w_gate, pitch_gate, H, K);
    o.add(w_up, pitch_up, H, K);
    const bool keep = images && type == LDN_F32;
    const size_t operands = keep ? 0 : o.bytes;
    Scratch scratch;
    r = scratch.take(st, operands + gated_tiles_scratch(GatedForm::Forward, rows, H, K, type, ctx));
    if (r == kOk) r = o.launch(keep ? static_cast<char*>(images) : scratch.base, ctx, st);
    if (r != kOk) return r;
    TileArgs t = {};
    t.M = rows;
    t.N = H;
    t.b_gate = b_gate; t.b_up = b_up; t.wide = a.wide; t.activation = activation;
    t.out0 = y; t.out1 = g; t.out2 = u;
    t.pitch = H; t.pitch_saved = pitch_saved;
    return launch_gated_tiles(GatedForm::Forward, t, K, o.images[0], o.images[1], o.images[2], type, scratch.base + operands, scratch.status,
                              ctx, st);
}

extern "C" LDN_API int ldn_gated_linear_backward(const void* grad_y, const void* x, long long pitch, long long rows, int K, int H, int type,
                                                 const void* w_gate, long long pitch_gate, const void* w_up, long long pitch_up, const float* g,
                                                 const float* u, long long pitch_saved, const void* images, int activation, void* grad_x, void* grad_w_gate,
                                                 void* grad_w_up, void* grad_b_gate, void* grad_b_up, int param_type, ldn_stream_t stream) {
    if (!gated_fits(rows, K, H, type, param_type, grad_b_gate, grad_b_up, activation, pitch_gate, pitch_up) || !grad_w_gate != !grad_w_up ||
        pitch_saved < H || pitch_saved % 16)
        return kBadArgument;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool wide = param_type == LDN_F32;
    const int size = size_of(type), param_size = wide ? 4 : size;
    int r = kOk;
    if (rows == 0) {
        const size_t weights = static_cast<size_t>(H) * K * size, bias = static_cast<size_t>(H) * param_size;
        for (void* p : {grad_w_gate, grad_w_up})
            if (p && r == kOk) r = cuda_status(cudaMemsetAsync(p, 0, weights, st));
        for (void* p : {grad_b_gate, grad_b_up})
            if (p && r == kOk) r = cuda_status(cudaMemsetAsync(p, 0, bias, st));
        return r;
    }
    if (!grad_y || !g || !u || !on32(g) || !on32(u) || (grad_x && (!w_gate || !w_up)) || (grad_w_gate && !x)) return kBadArgument;
    const DeviceCtx* ctx;
    if ((r = get_device_ctx(&ctx)) != kOk) return r;
    Operands o{type};
    const bool kept = images && type == LDN_F32;  // (all three, as the forward pass made them)
    const int at_x = grad_w_gate || kept ? o.add(x, pitch, rows, K) : 0;
    const int at_gate = grad_x || kept ? o.add(w_gate, pitch_gate, H, K) : 0, at_up = grad_x || kept ? o.add(w_up, pitch_up, H, K) : 0;
    if (kept) o.found(static_cast<char*>(const_cast<void*>(images)));
    const int parts = type == LDN_F32 ? 3 : 1;
    Images d;  // dg and du
    d.rows = rows;
    d.columns = H;
    d.pitch = padded8(H);
    d.count = 2 * parts;
    d.apart = rows * d.pitch;
    const int columns = (H + kGradColumns - 1) / kGradColumns;
    const long long most = (8LL * ctx->sm_count + columns - 1) / columns, needed = (rows + kGradRows - 1) / kGradRows;
    const int blocks = static_cast<int>(most < needed ? most : needed);
    const size_t d_bytes = pad256(static_cast<size_t>(d.count) * d.apart * 2), sum_bytes = pad256(static_cast<size_t>(blocks) * 2 * H * 4);
    size_t part_bytes = grad_x ? gated_tiles_scratch(GatedForm::GradRows, rows, K, H, type, ctx) : 0;
    const size_t more = grad_w_gate ? gated_tiles_scratch(GatedForm::GradWeights, H, K, static_cast<int>(rows), type, ctx) : 0;
    if (more > part_bytes) part_bytes = more;
    Scratch scratch;
    if ((r = scratch.take(st, d_bytes + sum_bytes + o.bytes + part_bytes)) != kOk) return r;
    d.base = scratch.base;
    float* sums = reinterpret_cast<float*>(scratch.base + d_bytes);
    char* left = scratch.base + d_bytes + sum_bytes;
    const bool biases = grad_b_gate || grad_b_up;
    const GradArgs ga = {grad_y, g, u, pitch_saved, rows, H, reinterpret_cast<unsigned short*>(scratch.base), d.pitch, d.apart,
                         biases ? sums : nullptr};
    r = with_type(type, [&](auto t) {
        using T = decltype(t);
        auto launch = [&](auto kernel) { return launch_after(kernel, dim3(columns, blocks), kGradLanes * kGradRows, 0, st, ga); };
        const int s = activation == LDN_SILU ? launch(gated_grad_kernel<T, LDN_SILU>) : activation == LDN_GELU ? launch(gated_grad_kernel<T, LDN_GELU>)
                    : activation == LDN_RELU ? launch(gated_grad_kernel<T, LDN_RELU>) : launch(gated_grad_kernel<T, LDN_SIGMOID>);
        if (s != kOk || !biases) return s;
        return launch_after(gated_fold_kernel<T>, dim3((H + kFoldColumns - 1) / kFoldColumns, 2), kFoldColumns * kFoldLanes, 0, st, sums, blocks,
                            H, wide, grad_b_gate, grad_b_up);
    });
    if (r == kOk) r = o.launch(left, ctx, st);
    left += o.bytes;
    TileArgs t = {};
    t.pitch = K;
    t.N = K;
    if (r == kOk && grad_x) {
        t.M = rows;
        t.out0 = grad_x;
        r = launch_gated_tiles(GatedForm::GradRows, t, H, d, o.images[at_gate], o.images[at_up], type, left, scratch.status, ctx, st);
    }
    if (r == kOk && grad_w_gate) {
        t.M = H;
        t.out0 = grad_w_gate;
        t.out1 = grad_w_up;
        r = launch_gated_tiles(GatedForm::GradWeights, t, static_cast<int>(rows), d, o.images[at_x], o.images[at_x], type, left, scratch.status,
                               ctx, st);
    }
    return r;
}
