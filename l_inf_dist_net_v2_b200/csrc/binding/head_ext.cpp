// The operators of a head (layer norm, dropout, the product in 8-bit integers) as functions of PyTorch tensors, with their
// autograd functions.  What is wrong with an argument raises before anything is launched; calls that other parts of PyTorch
// have to see (dispatch modes, the tracer, forward-mode tangents) are refused.
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <limits>

#include "ldn_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = c10::optional<Tensor>;

ldn_stream_t stream() { return reinterpret_cast<ldn_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }
void check(int status, const char* what) {
    TORCH_CHECK(status == 0, what, " failed with status ", status, ": ", ldn_status_string(status));
}
bool known(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
int type_of(at::ScalarType t) { return t == at::kFloat ? LDN_F32 : t == at::kHalf ? LDN_F16 : LDN_BF16; }
int type_of(const Tensor& t) { return type_of(t.scalar_type()); }

void plain(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.layout() == at::kStrided && t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch(), name,
                " must be plain memory");
    TORCH_CHECK(!t._fw_grad(0).defined(), name, " carries a forward-mode tangent, which this operator does not propagate");
}
void unobserved(const char* what) {
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::dispatch_mode_enabled(), what,
                " runs kernels of its own, which the tracer and dispatch modes do not see");
}
void activations(const Tensor& t, const char* name) {
    plain(t, name);
    TORCH_CHECK(known(t.scalar_type()), name, " must be float32, float16 or bfloat16, not ", t.scalar_type());
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1 && t.size(-1) <= std::numeric_limits<int>::max(), name, " has no rows: ", t.sizes());
}
void same_rows(const Tensor& t, const Tensor& x, const char* name) {
    activations(t, name);
    TORCH_CHECK(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device(), name,
                " must have the shape, type and device of x");
}
void parameter(const MaybeTensor& t, const Tensor& x, const char* name) {
    if (!t.has_value()) return;
    plain(*t, name);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), name, " must have one value per column");
    TORCH_CHECK((t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type()) && t->device() == x.device(), name,
                " must be float32 or of the type of x, on its device");
}
constexpr int64_t kMostColumns = std::numeric_limits<int>::max() - (1 << 22);
void row_fits(const Tensor& x) { TORCH_CHECK(x.size(-1) <= kMostColumns, "rows have at most ", kMostColumns, " elements, not ", x.size(-1)); }
void parameters(const MaybeTensor& weight, const MaybeTensor& bias, const Tensor& x, double eps) {
    row_fits(x);
    parameter(weight, x, "weight");
    parameter(bias, x, "bias");
    TORCH_CHECK(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(),
                "weight and bias must have one type");
    TORCH_CHECK(eps >= 0.0, "eps must not be negative");
}
int param_type(const MaybeTensor& weight, const MaybeTensor& bias) {
    return weight.has_value() ? type_of(*weight) : bias.has_value() ? type_of(*bias) : LDN_F32;
}
MaybeTensor whole(const MaybeTensor& t) { return t.has_value() ? MaybeTensor(t->contiguous()) : t; }
void* ptr(const MaybeTensor& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

// A tensor's rows: its memory as it is where rows are evenly spaced, else a copy
struct Rows {
    Tensor t;
    long long pitch, rows;
    int C;
};
Rows rows_of(const Tensor& x) {
    const int64_t C = x.size(-1), n = x.numel() / C;
    bool even = C == 1 || x.stride(-1) == 1;
    int64_t pitch = C, reach = -1;  // reach: the distance that the next dimension outwards has to have
    for (int64_t d = x.dim() - 2; even && d >= 0; --d) {
        if (x.size(d) == 1) continue;
        if (reach < 0) pitch = x.stride(d);
        else if (x.stride(d) != reach) even = false;
        reach = x.stride(d) * x.size(d);
    }
    if (even) return {x, pitch, n, static_cast<int>(C)};
    return {x.contiguous(), C, n, static_cast<int>(C)};
}
float* floats(const Tensor& t) { return t.data_ptr<float>(); }

// Seed, offset and device words of one call
struct Draw {
    double p;
    int64_t seed, offset;
    Tensor state;
    const unsigned long long* words() const {
        return state.defined() ? reinterpret_cast<const unsigned long long*>(state.data_ptr<int64_t>()) : nullptr;
    }
    unsigned long long seed64() const { return static_cast<unsigned long long>(seed); }
    unsigned long long offset64() const { return static_cast<unsigned long long>(offset); }
    MaybeTensor given() const { return state.defined() ? MaybeTensor(state) : c10::nullopt; }
    // (the device words of a later backward pass are those of now, whatever the caller draws next)
    void keep(AutogradContext* ctx) const {
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        if (state.defined()) ctx->saved_data["state"] = state;
    }
    static Draw kept(AutogradContext* ctx) {
        const auto state = ctx->saved_data.find("state");
        return {ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt(),
                state == ctx->saved_data.end() ? Tensor() : state->second.toTensor()};
    }
};
Draw draw_of(double p, int64_t seed, int64_t offset, const MaybeTensor& state, const Tensor& x, bool keep) {
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "p must be a probability, not ", p);
    if (!state.has_value()) return {p, seed, offset, Tensor()};
    plain(*state, "seed");
    TORCH_CHECK(state->scalar_type() == at::kLong && state->dim() == 1 && state->size(0) == 2 && state->device() == x.device(),
                "a seed on the device must be two int64 values, seed and offset, on the device of x");
    return {p, seed, offset, keep ? state->clone(at::MemoryFormat::Contiguous) : state->contiguous()};
}

void once(const variable_list& grads, const char* what) {
    for (const Tensor& g : grads)
        TORCH_CHECK(!(at::GradMode::is_enabled() && g.defined() && g.requires_grad()), "the gradient of ", what,
                    " cannot be differentiated again");
}

// A gradient that is one once only: it goes on as a function of `of`, so that whoever differentiates it again, wherever the
// differentiation comes from, is told that there is no such derivative (without it, it would pass for a constant).
struct OnceFn : public torch::autograd::Function<OnceFn> {
    static Tensor forward(AutogradContext* ctx, Tensor grad, Tensor of, std::string what) {
        ctx->saved_data["what"] = what;
        return grad.detach();
    }
    static variable_list backward(AutogradContext* ctx, variable_list) {
        TORCH_CHECK(false, "the gradient of ", ctx->saved_data["what"].toStringRef(), " cannot be differentiated again");
        return {};
    }
};
Tensor once_of(const Tensor& grad, std::initializer_list<const Tensor*> depends_on, const char* what) {
    if (grad.defined() && at::GradMode::is_enabled())
        for (const Tensor* t : depends_on)
            if (t->defined() && t->requires_grad()) return OnceFn::apply(grad, *t, std::string(what));
    return grad;
}

// ---- layer norm ---------------------------------------------------------------------------------------------------------------
void norm_forward(const Rows& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, Tensor& y, float* stats) {
    check(ldn_layer_norm(x.t.data_ptr(), x.pitch, x.rows, x.C, type_of(x.t), ptr(weight), ptr(bias), param_type(weight, bias),
                         static_cast<float>(eps), y.data_ptr(), stats, stats ? stats + x.rows : nullptr, stream()),
          "layer_norm");
}

struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
    static Tensor forward(AutogradContext* ctx, Tensor x, MaybeTensor weight, MaybeTensor bias, double eps) {
        const c10::cuda::CUDAGuard guard(x.device());
        const MaybeTensor w = whole(weight), b = whole(bias);
        const Rows rows = rows_of(x);
        Tensor y = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
        Tensor stats = at::empty({2, rows.rows}, x.options().dtype(at::kFloat));
        norm_forward(rows, w, b, eps, y, floats(stats));
        ctx->saved_data["param_type"] = param_type(weight, bias);
        ctx->saved_data["bias"] = bias.has_value();
        ctx->save_for_backward({x, w.has_value() ? *w : Tensor(), stats});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once(grads, "layer_norm");
        variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
        const c10::cuda::CUDAGuard guard(x.device());
        const Rows rows = rows_of(x);
        const Tensor g = grads[0].contiguous();
        const int params = static_cast<int>(ctx->saved_data["param_type"].toInt());
        const auto as_param = x.options().dtype(params == LDN_F32 ? at::kFloat : x.scalar_type());
        Tensor gx, gw, gb;
        int edge = 0;  // (absent parameters have none)
        if (ctx->needs_input_grad(edge++)) gx = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
        if (w.defined() && ctx->needs_input_grad(edge++)) gw = at::empty({rows.C}, as_param);
        if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(edge++)) gb = at::empty({rows.C}, as_param);
        check(ldn_layer_norm_backward(g.data_ptr(), rows.t.data_ptr(), rows.pitch, rows.rows, rows.C, type_of(x), floats(stats),
                                      floats(stats) + rows.rows, w.defined() ? w.data_ptr() : nullptr, params, ptr(gx), ptr(gw),
                                      ptr(gb), stream()),
              "layer_norm_backward");
        return {once_of(gx, {&x, &w}, "layer_norm"), once_of(gw, {&x}, "layer_norm"), gb, Tensor()};
    }
};

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t && t->requires_grad()) return true;
    return false;
}
const Tensor* at_of(const MaybeTensor& t) { return t.has_value() ? &*t : nullptr; }

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
    unobserved("layer_norm");
    activations(x, "x");
    parameters(weight, bias, x, eps);
    if (wants_grad({&x, at_of(weight), at_of(bias)})) return LayerNormFn::apply(x, weight, bias, eps);
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
    norm_forward(rows_of(x), whole(weight), whole(bias), eps, y, nullptr);
    return y;
}

// ---- dropout ------------------------------------------------------------------------------------------------------------------
Tensor drop(const Tensor& x, const MaybeTensor& residual, const Draw& d) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows rows = rows_of(x);
    const Rows onto = residual.has_value() ? rows_of(*residual) : Rows{Tensor(), 0, 0, 0};
    Tensor out = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
    check(ldn_dropout(rows.t.data_ptr(), rows.pitch, onto.t.defined() ? onto.t.data_ptr() : nullptr, onto.pitch, rows.rows, rows.C,
                      type_of(x), d.p, d.seed64(), d.offset64(), d.words(), out.data_ptr(), stream()),
          "dropout");
    return out;
}

struct DropoutFn : public torch::autograd::Function<DropoutFn> {
    static Tensor forward(AutogradContext* ctx, Tensor x, MaybeTensor residual, double p, int64_t seed, int64_t offset,
                          MaybeTensor state) {
        const Draw d{p, seed, offset, state.has_value() ? *state : Tensor()};
        d.keep(ctx);
        ctx->saved_data["residual"] = residual.has_value();
        return drop(x, residual, d);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Draw d = Draw::kept(ctx);
        Tensor gx;
        if (ctx->needs_input_grad(0)) {  // (linear, so the gradient of the gradient is the operator once more)
            activations(grads[0], "grad");
            gx = wants_grad({&grads[0]}) ? DropoutFn::apply(grads[0], c10::nullopt, d.p, d.seed, d.offset, d.given())
                                         : drop(grads[0], c10::nullopt, d);
        }
        const bool onto = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
        return {gx, onto ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor& x, double p, int64_t seed, int64_t offset, const MaybeTensor& state, const MaybeTensor& residual) {
    unobserved("dropout");
    activations(x, "x");
    if (residual.has_value()) same_rows(*residual, x, "residual");
    const bool grad = wants_grad({&x, at_of(residual)});
    const Draw d = draw_of(p, seed, offset, state, x, grad);
    return grad ? DropoutFn::apply(x, residual, p, seed, offset, d.given()) : drop(x, residual, d);
}

// ---- both, on a residual stream -------------------------------------------------------------------------------------------------
void joined_forward(const Tensor& x, const Tensor& residual, const MaybeTensor& w, const MaybeTensor& b, double eps, const Draw& d,
                    Tensor& h, Tensor& y, float* stats) {
    const Rows rows = rows_of(x), onto = rows_of(residual);
    check(ldn_dropout_add_layer_norm(rows.t.data_ptr(), rows.pitch, onto.t.data_ptr(), onto.pitch, rows.rows, rows.C, type_of(x),
                                     ptr(w), ptr(b), param_type(w, b), static_cast<float>(eps), d.p, d.seed64(), d.offset64(),
                                     d.words(), h.data_ptr(), y.data_ptr(), stats, stats ? stats + rows.rows : nullptr, stream()),
          "dropout_add_layer_norm");
}

struct DropoutAddNormFn : public torch::autograd::Function<DropoutAddNormFn> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor residual, MaybeTensor weight, MaybeTensor bias, double eps,
                                 double p, int64_t seed, int64_t offset, MaybeTensor state) {
        const c10::cuda::CUDAGuard guard(x.device());
        const Draw d{p, seed, offset, state.has_value() ? *state : Tensor()};
        const MaybeTensor w = whole(weight), b = whole(bias);
        Tensor y = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
        Tensor h = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
        Tensor stats = at::empty({2, x.numel() / x.size(-1)}, x.options().dtype(at::kFloat));
        joined_forward(x, residual, w, b, eps, d, h, y, floats(stats));
        ctx->set_materialize_grads(false);
        d.keep(ctx);
        ctx->saved_data["param_type"] = param_type(weight, bias);
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["rows"] = x.requires_grad() || residual.requires_grad();
        ctx->save_for_backward({h, w.has_value() ? *w : Tensor(), stats});
        return {y, h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return variable_list(9);
        once(grads, "dropout_add_layer_norm");
        variable_list saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &w = saved[1], &stats = saved[2];
        const c10::cuda::CUDAGuard guard(h.device());
        const Draw d = Draw::kept(ctx);
        const int64_t C = h.size(-1), rows = h.numel() / C;
        const Tensor gy = grads[0].defined() ? grads[0].contiguous() : at::zeros_like(h);
        const Tensor gh = grads[1].defined() ? grads[1].contiguous() : Tensor();
        const int params = static_cast<int>(ctx->saved_data["param_type"].toInt());
        const auto as_param = h.options().dtype(params == LDN_F32 ? at::kFloat : h.scalar_type());
        Tensor gx, gr, gw, gb;
        int edge = 0;  // (absent parameters have none)
        if (ctx->needs_input_grad(edge++)) gx = at::empty_like(h);
        if (ctx->needs_input_grad(edge++)) gr = at::empty_like(h);
        if (w.defined() && ctx->needs_input_grad(edge++)) gw = at::empty({C}, as_param);
        if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(edge++)) gb = at::empty({C}, as_param);
        check(ldn_dropout_add_layer_norm_backward(gy.data_ptr(), ptr(gh), h.data_ptr(), rows, static_cast<int>(C), type_of(h),
                                                  floats(stats), floats(stats) + rows, w.defined() ? w.data_ptr() : nullptr,
                                                  params, d.p, d.seed64(), d.offset64(), d.words(), ptr(gx), ptr(gr), ptr(gw),
                                                  ptr(gb), stream()),
              "dropout_add_layer_norm_backward");
        const char* what = "dropout_add_layer_norm";
        if (ctx->saved_data["rows"].toBool()) gw = once_of(gw, {&h}, what);  // (h has a gradient if the weight alone has one, too)
        return {once_of(gx, {&h, &w}, what), once_of(gr, {&h, &w}, what), gw, gb, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const MaybeTensor& weight,
                                                  const MaybeTensor& bias, double p, int64_t seed, int64_t offset,
                                                  const MaybeTensor& state, double eps) {
    unobserved("dropout_add_layer_norm");
    activations(x, "x");
    same_rows(residual, x, "residual");
    parameters(weight, bias, x, eps);
    const bool grad = wants_grad({&x, &residual, at_of(weight), at_of(bias)});
    const Draw d = draw_of(p, seed, offset, state, x, grad);
    if (grad) {
        variable_list out = DropoutAddNormFn::apply(x, residual, weight, bias, eps, p, seed, offset, d.given());
        return std::make_tuple(out[0], out[1]);
    }
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous), h = at::empty_like(y);
    joined_forward(x, residual, whole(weight), whole(bias), eps, d, h, y, nullptr);
    return std::make_tuple(y, h);
}

// ---- 8-bit integers -------------------------------------------------------------------------------------------------------------
// Integers of a tensor's shape whose rows start at multiples of 16 bytes
Tensor integers(const Tensor& x) {
    const int64_t C = x.size(-1), pitch = (C + 15) / 16 * 16;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = pitch;
    return at::empty(shape, x.options().dtype(at::kChar)).narrow(-1, 0, C);
}
Tensor scales(const Tensor& x) { return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat)); }
long long padded(long long C) { return (C + 15) / 16 * 16; }

void answers_only(bool grad, const char* what) { TORCH_CHECK(!grad, what, " has no gradient: call it under torch.no_grad()"); }

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
    unobserved("quantize_rows");
    activations(x, "x");
    row_fits(x);
    answers_only(wants_grad({&x}), "quantize_rows");
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows rows = rows_of(x);
    Tensor q = integers(x), scale = scales(x);
    check(ldn_quantize_rows(rows.t.data_ptr(), rows.pitch, rows.rows, rows.C, type_of(x),
                            static_cast<signed char*>(q.data_ptr()), padded(rows.C), floats(scale), stream()),
          "quantize_rows");
    return std::make_tuple(q, scale);
}

std::tuple<Tensor, Tensor> layer_norm_quantized(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
    unobserved("layer_norm_quantized");
    activations(x, "x");
    parameters(weight, bias, x, eps);
    answers_only(wants_grad({&x, at_of(weight), at_of(bias)}), "layer_norm_quantized");
    const c10::cuda::CUDAGuard guard(x.device());
    const MaybeTensor w = whole(weight), b = whole(bias);
    const Rows rows = rows_of(x);
    Tensor q = integers(x), scale = scales(x);
    check(ldn_layer_norm_quantized(rows.t.data_ptr(), rows.pitch, rows.rows, rows.C, type_of(x), ptr(w), ptr(b), param_type(w, b),
                                   static_cast<float>(eps), static_cast<signed char*>(q.data_ptr()), padded(rows.C), floats(scale),
                                   stream()),
          "layer_norm_quantized");
    return std::make_tuple(q, scale);
}

void bytes(const Tensor& t, const char* name) {
    plain(t, name);
    TORCH_CHECK(t.scalar_type() == at::kChar, name, " must be int8, not ", t.scalar_type());
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, name, " has no rows: ", t.sizes());
}
// x: rows in floating point, or integers with x_scale
Tensor int8_linear(const Tensor& x, const MaybeTensor& x_scale, const Tensor& weight, const Tensor& weight_scale,
                   const MaybeTensor& bias, int64_t activation, const c10::optional<at::ScalarType>& out_type) {
    unobserved("int8_linear");
    if (x_scale.has_value()) bytes(x, "x");
    else activations(x, "x");
    bytes(weight, "weight");
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == x.size(-1), "weight must be (outputs, ", x.size(-1), "), not ", weight.sizes());
    TORCH_CHECK(weight.size(0) >= 1 && weight.size(0) <= kMostColumns, "weight must have 1 to ", kMostColumns, " outputs");
    TORCH_CHECK(weight.size(1) <= 131071, "sums of ", weight.size(1), " products do not fit 32 bits: at most 131071 do");
    TORCH_CHECK(weight.device() == x.device(), "weight must be on the device of x");
    for (const Tensor* t : {&weight_scale, at_of(bias), at_of(x_scale)})
        if (t) {
            plain(*t, "scale or bias");
            TORCH_CHECK(t->scalar_type() == at::kFloat && t->device() == x.device(), "scales and bias must be float32 on the device of x");
        }
    TORCH_CHECK(weight_scale.dim() == 1 && weight_scale.size(0) == weight.size(0), "weight needs one scale per output");
    TORCH_CHECK(!bias.has_value() || (bias->dim() == 1 && bias->size(0) == weight.size(0)), "bias must have one value per output");
    TORCH_CHECK(!x_scale.has_value() || x_scale->sizes() == x.sizes().slice(0, x.dim() - 1), "x needs one scale per row");
    TORCH_CHECK(!out_type.has_value() || known(*out_type), "out_dtype must be float32, float16 or bfloat16");
    answers_only(wants_grad({&x, &weight_scale, at_of(bias), at_of(x_scale)}), "int8_linear");
    const at::ScalarType type = out_type.has_value() ? *out_type : x_scale.has_value() ? at::kFloat : x.scalar_type();
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows rows = rows_of(x), w = rows_of(weight);
    const Tensor ws = weight_scale.contiguous();
    const MaybeTensor b = whole(bias);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = weight.size(0);
    Tensor out = at::empty(shape, x.options().dtype(type));
    const signed char* wq = static_cast<const signed char*>(w.t.data_ptr());
    const int N = static_cast<int>(weight.size(0));
    TORCH_CHECK(w.rows == 1 || w.pitch >= w.C, "weight's rows must not overlap");
    const long long pitch_w = w.rows == 1 ? padded(w.C) : w.pitch;
    const float* fb = static_cast<const float*>(ptr(b));
    if (x_scale.has_value()) {
        TORCH_CHECK(rows.rows <= 1 || rows.pitch >= rows.C, "x's rows must not overlap");
        const Tensor xs = x_scale->contiguous();
        check(ldn_int8_linear(static_cast<const signed char*>(rows.t.data_ptr()), rows.rows <= 1 ? padded(rows.C) : rows.pitch,
                              floats(xs), wq, pitch_w, floats(ws), fb, rows.rows, N, rows.C, static_cast<int>(activation),
                              out.data_ptr(), type_of(type), stream()),
              "int8_linear");
    } else {
        check(ldn_int8_linear_float(rows.t.data_ptr(), rows.pitch, type_of(x), wq, pitch_w, floats(ws), fb, rows.rows, N, rows.C,
                                    static_cast<int>(activation), out.data_ptr(), type_of(type), stream()),
              "int8_linear");
    }
    return out;
}

}  // namespace

void register_head(pybind11::module& m) {
    m.def("layer_norm", &layer_norm);
    m.def("dropout", &dropout);
    m.def("dropout_add_layer_norm", &dropout_add_layer_norm);
    m.def("quantize_rows", &quantize_rows);
    m.def("layer_norm_quantized", &layer_norm_quantized);
    m.def("int8_linear", &int8_linear);
}
