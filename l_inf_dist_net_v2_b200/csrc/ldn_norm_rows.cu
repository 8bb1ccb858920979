// Layer norm forward (and rows as integers) with the row in registers: one read of the row, two sums over it (the mean, then the
// squares of what is left), one write.  Bound by memory: what a call cannot do without is x and y once.
#include "ldn_norm.cuh"
#include "ldn_rows.cuh"

namespace ldn {
namespace {

// 32 elements per thread, so that 128 registers hold them beside the rest: rows of up to 16384
constexpr int kMostThreads = 512;
template <class T>
constexpr int kMostItems = 32 / kPiece<T>;

template <class T, Form F, int ITEMS, bool GROUP, bool SHIFT>
__global__ void __launch_bounds__(GROUP ? kGroupThreads : kMostThreads) norm_registers_kernel(NormArgs a, int lanes) {
    stream_order_begin();
    constexpr int V = kPiece<T>;
    __shared__ float slots[128];
    RowSum reduce{lanes, slots, 0};
    Generator gen;
    if constexpr (F == Form::Joined) gen = generator_of(a.drop);
    const int lane = GROUP ? threadIdx.x & (lanes - 1) : threadIdx.x;
    const int per_block = GROUP ? kGroupThreads / lanes : 1;
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    const float inv_C = 1.0f / a.C;
    // (a warp's groups take part in its shuffles whether they have a row or not)
    for (long long first = static_cast<long long>(blockIdx.x) * per_block; first < a.rows; first += step) {
        const long long row = GROUP ? first + threadIdx.x / lanes : first;
        const bool live = !GROUP || row < a.rows;
        const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.pitch;
        const long long at = (live ? row : 0) * a.C;
        const int C = live ? a.C : 0, shift = SHIFT ? shift_of(x) : 0;
        float v[ITEMS][V];
        {
            uint4 raw[ITEMS], onto[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) raw[i] = load_piece<T, SHIFT>(x, (lane + i * lanes) * V - shift, C);
            if constexpr (F == Form::Joined) {
                const T* res = static_cast<const T*>(a.residual) + (live ? row : 0) * a.pitch_residual;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) onto[i] = load_piece<T, SHIFT>(res, (lane + i * lanes) * V - shift, C);
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                unpack<T>(raw[i], v[i]);
                if constexpr (F == Form::Joined) {
                    const int c0 = (lane + i * lanes) * V - shift;
                    float r[V];
                    unpack<T>(onto[i], r);
                    // (pieces start at multiples of four elements of the whole tensor)
#pragma unroll
                    for (int e = 0; e < V; e += 4) {
                        const uint4 w = random_words(gen, static_cast<unsigned long long>(at + c0 + e) >> 2);
                        v[i][e] = __fadd_rn(r[e], dropped(a.drop, w.x, v[i][e]));
                        v[i][e + 1] = __fadd_rn(r[e + 1], dropped(a.drop, w.y, v[i][e + 1]));
                        v[i][e + 2] = __fadd_rn(r[e + 2], dropped(a.drop, w.z, v[i][e + 2]));
                        v[i][e + 3] = __fadd_rn(r[e + 3], dropped(a.drop, w.w, v[i][e + 3]));
                    }
                    const uint4 h = pack<T>(v[i]);
                    store_piece<T, SHIFT>(static_cast<T*>(a.h) + at, c0, C, h);
                    unpack<T>(h, v[i]);
                    if (SHIFT) {  // (dropout of nothing is the residual's nothing: 0)
#pragma unroll
                        for (int e = 0; e < V; ++e) v[i][e] = in_row<SHIFT>(c0, e, C) ? v[i][e] : 0.0f;
                    }
                }
            }
        }
        if constexpr (F != Form::Quantised) {
            float s[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) s[0] += v[i][e];
            reduce.template sum<1, GROUP>(s);
            const float mean = s[0] * inv_C;
            s[0] = 0.0f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c0 = (lane + i * lanes) * V - shift;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    v[i][e] = in_row<SHIFT>(c0, e, C) ? v[i][e] - mean : 0.0f;
                    s[0] += v[i][e] * v[i][e];
                }
            }
            reduce.template sum<1, GROUP>(s);
            const float rstd = 1.0f / sqrtf(s[0] * inv_C + a.eps);
            if (lane == 0 && live && a.mean) {
                a.mean[row] = mean;
                a.rstd[row] = rstd;
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c0 = (lane + i * lanes) * V - shift;
                float w[V], b[V];
                load_params<T, SHIFT>(a.weight, a.wide, c0, C, 1.0f, w);
                load_params<T, SHIFT>(a.bias, a.wide, c0, C, 0.0f, b);
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = fmaf(v[i][e] * rstd, w[e], b[e]);
                if constexpr (F != Form::Integers) store_piece<T, SHIFT>(static_cast<T*>(a.y) + at, c0, C, pack<T>(v[i]));
            }
        }
        if constexpr (F == Form::Integers || F == Form::Quantised) {
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) top = max(top, magnitude(v[i][e]));
            const float size = step_of(reduce.template largest<GROUP>(top)), inverse = 1.0f / size;
            if (lane == 0 && live) a.scale[row] = size;
            signed char* q = a.q + row * a.pitch_q;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c0 = (lane + i * lanes) * V - shift;
                unsigned word[V / 4];
#pragma unroll
                for (int e = 0; e < V; e += 4)
                    word[e / 4] = (steps(v[i][e], inverse) & 255) | (steps(v[i][e + 1], inverse) & 255) << 8 |
                                  (steps(v[i][e + 2], inverse) & 255) << 16 | static_cast<unsigned>(steps(v[i][e + 3], inverse)) << 24;
                if (!SHIFT) {  // (the integers' rows start at multiples of 16 bytes then)
                    if (c0 < C) {
                        if constexpr (V == 8) *reinterpret_cast<uint2*>(q + c0) = make_uint2(word[0], word[1]);
                        else *reinterpret_cast<unsigned*>(q + c0) = word[0];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (in_row<SHIFT>(c0, e, C)) q[c0 + e] = static_cast<signed char>(word[e / 4] >> 8 * (e % 4));
                }
            }
        }
    }
}

template <class T, Form F, int ITEMS, bool GROUP, bool SHIFT>
int launch(const NormArgs& a, const RowPlan& p, const DeviceCtx* ctx, cudaStream_t st) {
    static std::atomic<int> resident[64][33];  // blocks per SM by warps
    std::atomic<int>& known = resident[ctx->device][p.threads / 32];
    int per_sm = known.load(std::memory_order_acquire);
    if (per_sm == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, norm_registers_kernel<T, F, ITEMS, GROUP, SHIFT>, p.threads, 0) !=
                cudaSuccess || per_sm < 1) {
            cudaGetLastError();
            per_sm = 1;
        }
        known.store(per_sm, std::memory_order_release);
    }
    const long long most = static_cast<long long>(per_sm) * ctx->sm_count, blocks = (a.rows + p.rows_per_block() - 1) / p.rows_per_block();
    return launch_after(norm_registers_kernel<T, F, ITEMS, GROUP, SHIFT>, static_cast<unsigned>(blocks < most ? blocks : most), p.threads,
                        0, st, a, p.lanes);
}
template <class T, Form F, int ITEMS>
int launch(const NormArgs& a, const RowPlan& p, const DeviceCtx* ctx, cudaStream_t st) {
    if (p.group) return p.shift ? launch<T, F, ITEMS, true, true>(a, p, ctx, st) : launch<T, F, ITEMS, true, false>(a, p, ctx, st);
    return p.shift ? launch<T, F, ITEMS, false, true>(a, p, ctx, st) : launch<T, F, ITEMS, false, false>(a, p, ctx, st);
}
template <class T, Form F>
int launch(const NormArgs& a, const RowPlan& p, const DeviceCtx* ctx, cudaStream_t st) {
    switch (p.items) {
        case 1: return launch<T, F, 1>(a, p, ctx, st);
        case 2: return launch<T, F, 2>(a, p, ctx, st);
        case 4: return launch<T, F, 4>(a, p, ctx, st);
        default: return launch<T, F, kMostItems<T>>(a, p, ctx, st);
    }
}

}  // namespace

bool norm_in_registers(Form form, const NormArgs& a, int type, const DeviceCtx* ctx, cudaStream_t st, int* status) {
    const int size = size_of(type);
    bool aligned = on16(a.x) && on16(a.y) && on16(a.h) && on16(a.residual);  // (the ones that the form has not are null)
    bool match = rows_match(size, a.C, a.pitch, aligned);
    if (form == Form::Joined) match = match && rows_match(size, a.C, a.pitch_residual, aligned);
    bool shift = rows_shift(size, a.C) || !on16(a.weight) || !on16(a.bias);
    if (form == Form::Integers || form == Form::Quantised) {
        // nothing has to match x but the integers, which are stored one by one where they do not
        match = (reinterpret_cast<uintptr_t>(a.x) & (size - 1)) == 0;
        shift = shift || !on16(a.x) || a.pitch * size % 16 != 0 || !on16(a.q) || a.pitch_q % 16 != 0;
    }
    RowPlan p;
    if (!match || !plan_rows(a.C, 16 / size, shift, 2 * size, kMostThreads, 1, &p)) return false;
    *status = with_type(type, [&](auto t) {
        using T = decltype(t);
        switch (form) {
            case Form::Plain: return launch<T, Form::Plain>(a, p, ctx, st);
            case Form::Joined: return launch<T, Form::Joined>(a, p, ctx, st);
            case Form::Integers: return launch<T, Form::Integers>(a, p, ctx, st);
            default: return launch<T, Form::Quantised>(a, p, ctx, st);
        }
    });
    return true;
}

}  // namespace ldn
