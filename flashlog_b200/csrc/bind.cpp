// bind.cpp -- the relation-attention operators on torch tensors.
//
// Checks, allocation and autograd around the C ABI of libflashlog_b200.so.  In
// Python they cost 60 to 80 us of a training call whose kernels take 40.
// Everything runs on the current stream of the tensors' device; workspaces are
// allocated by the call (a captured call's belong to its graph).
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <limits>
#include <optional>
#include <vector>

#include "../../include/flashlog_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxColumns = 65536, kMaxHistory = 65535;

#define FL_VALUE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

std::string shape_text(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

int dtype_of(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return FL_F32;
        case at::kHalf: return FL_F16;
        case at::kBFloat16: return FL_BF16;
        default: return -1;
    }
}

bool given(const OptTensor &t) { return t.has_value() && t->defined(); }
template <typename T = void>
T *ptr(const OptTensor &t) {
    return given(t) ? static_cast<T *>(t->data_ptr()) : nullptr;
}
template <typename T = void>
T *ptr(const Tensor &t) {
    return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}

void check(int rc, const char *what) {
    if (rc == FL_OK) return;
    if (rc == FL_EINVAL) FL_VALUE(false, what, ": ", fl_last_error());
    TORCH_CHECK(false, what, ": ", fl_last_error(), " (status ", rc, ")");
}

// One CUDA device for all tensors of a call.
struct Devices {
    const char *what;
    const Tensor *first = nullptr;
    void add(const Tensor &t) {
        if (!t.defined()) return;
        FL_VALUE(t.is_cuda(), "flashlog_b200 runs on CUDA tensors only (no CPU fallback)");
        if (first == nullptr) first = &t;
        else FL_VALUE(t.device() == first->device(), what, ": tensors on ", first->device(), " and ", t.device());
    }
    void add(const OptTensor &t) {
        if (given(t)) add(*t);
    }
};
struct OnDevice {
    c10::cuda::OptionalCUDAGuard guard;
    fl_stream_t stream;
    explicit OnDevice(const Tensor &t) {
        guard.set_device(t.device());
        stream = reinterpret_cast<fl_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
    }
};

// [rows, cols] lines that the library can address: unit inner stride, rows at least a row apart.
Tensor lines(const Tensor &t) {
    if (t.is_contiguous() || (t.stride(1) == 1 && (t.stride(0) >= t.size(1) || t.size(0) <= 1))) return t;
    return t.contiguous();
}
int64_t ld(const Tensor &t) { return std::max(t.stride(0), t.size(1)); }
Tensor workspace(size_t bytes, const Tensor &like) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}
bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor &t) { return given(t) && t->requires_grad(); }

// Autograd's note that a kernel wrote into a tensor that it may have saved.
void written(const Tensor &t) {
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

// Forward-mode derivatives are not there: an error, not a result without its tangent.
void no_tangent(const char *what, std::initializer_list<OptTensor> tensors) {
    for (const OptTensor &t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!given(t) || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}

// Passes a gradient on; differentiating it again is an error, not a silent zero.
// The tensors after it are what it was made of.
struct Once : torch::autograd::Function<Once> {
    static Tensor forward(AutogradContext *, const Tensor &grad, const OptTensor &, const OptTensor &, const OptTensor &,
                          const OptTensor &) {
        return grad.view_as(grad);
    }
    static variable_list backward(AutogradContext *, variable_list) {
        TORCH_CHECK(false, "flashlog_b200 attention operators are differentiable once");
    }
};
Tensor once(const Tensor &grad, const OptTensor &gy, const OptTensor &a, const OptTensor &b = std::nullopt,
            const OptTensor &c = std::nullopt) {
    if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
    if (!(wants_grad(gy) || wants_grad(a) || wants_grad(b) || wants_grad(c))) return grad;
    return Once::apply(grad, gy, a, b, c);
}

// ---- the head --------------------------------------------------------------------
fl_linear linear_params(const Tensor &x, const Tensor &w, const OptTensor &bias, const OptTensor &residual, int64_t act) {
    fl_linear p{};
    p.x = ptr(x);
    p.w = ptr(w);
    p.bias = ptr(bias);
    p.residual = ptr(residual);
    p.ld_x = ld(x);
    p.ld_w = ld(w);
    p.ld_res = given(residual) ? ld(*residual) : 0;
    p.rows = x.size(0);
    p.n = w.size(0);
    p.k = w.size(1);
    p.dtype = dtype_of(x);
    p.act = static_cast<int>(act);
    return p;
}

// (y, z) of 2-D tensors; z (the fp32 pre-activation) with want_z and an activation only
std::tuple<Tensor, Tensor> linear_forward(const Tensor &x0, const Tensor &w0, const OptTensor &bias0,
                                          const OptTensor &residual0, int64_t act, bool want_z, const OptTensor &out) {
    Devices d{"linear"};
    d.add(x0);
    d.add(w0);
    d.add(bias0);
    d.add(residual0);
    d.add(out);
    const Tensor x = lines(x0), w = lines(w0);
    const OptTensor bias = given(bias0) ? OptTensor(bias0->contiguous()) : bias0;
    const OptTensor residual = given(residual0) ? OptTensor(lines(*residual0)) : residual0;
    const int64_t rows = x.size(0), n = w.size(0);
    Tensor y = given(out) ? *out : at::empty({rows, n}, x.options());
    Tensor z = want_z && act != FL_ACT_NONE ? at::empty({rows, n}, x.options().dtype(at::kFloat)) : Tensor();
    if (rows == 0) return {y, z};
    const fl_linear p = linear_params(x, w, bias, residual, act);
    OnDevice on(x);
    const size_t bytes = fl_linear_workspace(rows, n, p.k, p.dtype);
    const Tensor ws = workspace(bytes, x);
    check(fl_linear_forward(&p, ptr(y), n, ptr<float>(z), ptr(ws), bytes, on.stream), "linear");
    if (given(out)) written(y);
    return {y, z};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor &x0, const Tensor &w0, const OptTensor &z, const Tensor &gy0,
                                                   int64_t act, bool want_x, bool want_w, bool want_bias) {
    Devices d{"linear backward"};
    d.add(x0);
    d.add(w0);
    d.add(z);
    d.add(gy0);
    const Tensor x = lines(x0), w = lines(w0), gy = lines(gy0);
    const int64_t rows = x.size(0), n = w.size(0), k = w.size(1);
    Tensor dx = want_x ? at::empty({rows, k}, x.options()) : Tensor();
    Tensor dw = want_w ? at::empty({n, k}, x.options()) : Tensor();
    Tensor db = want_bias ? at::empty({n}, x.options()) : Tensor();
    const fl_linear p = linear_params(x, w, std::nullopt, std::nullopt, act);
    OnDevice on(x);
    const size_t bytes = fl_linear_backward_workspace(rows, n, k, p.dtype, p.act);
    const Tensor ws = workspace(bytes, x);
    check(fl_linear_backward(&p, ptr<float>(z), ptr(gy), ld(gy), ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, on.stream),
          "linear backward");
    return {dx, dw, db};
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &bias,
                          const OptTensor &residual, int64_t act) {
        auto [y, z] = linear_forward(x, w, bias, residual, act, true, std::nullopt);
        ctx->saved_data["act"] = act;
        ctx->saved_data["bias"] = given(bias);
        ctx->saved_data["residual"] = given(residual);
        // the gradients do not read the bias (it may change in place); with an activation they depend on it
        if (act != FL_ACT_NONE && wants_grad(bias)) ctx->saved_data["through_bias"] = *bias;
        ctx->save_for_backward({x, w, z});
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const bool bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
        // edges exist for the tensors that were given
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const bool want_bias = bias && ctx->needs_input_grad(2);
        const bool want_res = residual && ctx->needs_input_grad(bias ? 3 : 2);
        const Tensor gy = grads[0];
        variable_list out(5);
        if (!gy.defined()) return out;
        if (want_x || want_w || want_bias) {
            Tensor dx, dw, db;
            {
                at::AutoDispatchBelowADInplaceOrView below;
                std::tie(dx, dw, db) = linear_backward(saved[0], saved[1], saved[2], gy, ctx->saved_data["act"].toInt(),
                                                       want_x, want_w, want_bias);
            }
            const Tensor &x = saved[0], &w = saved[1];
            if (ctx->saved_data["act"].toInt() == FL_ACT_NONE) {
                out[0] = once(dx, gy, w);
                out[1] = once(dw, gy, x);
                out[2] = once(db, gy, std::nullopt);
            } else {  // act' at the pre-activation, which every input has a part in
                const auto it = ctx->saved_data.find("through_bias");
                const Tensor b = it == ctx->saved_data.end() ? Tensor() : it->second.toTensor();
                out[0] = once(dx, gy, x, w, b);
                out[1] = once(dw, gy, x, w, b);
                out[2] = once(db, gy, x, w, b);
            }
        }
        if (want_res) out[3] = gy;
        return out;
    }
};

Tensor linear(const Tensor &x, const Tensor &w, const OptTensor &bias, const OptTensor &residual, int64_t act) {
    const int dt = dtype_of(x);
    FL_VALUE(dt >= 0, "linear takes float32, float16 or bfloat16 tensors, got ", x.scalar_type());
    FL_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1), "linear: x [..., k] and weight [n, k], got ",
             shape_text(x.sizes()), " and ", shape_text(w.sizes()));
    const int64_t n = w.size(0), k = w.size(1);
    FL_VALUE(n > 0 && k > 0, "linear: weight must not be empty");
    FL_VALUE(w.scalar_type() == x.scalar_type(), "linear: tensors of one dtype, got ", x.scalar_type(), " and ", w.scalar_type());
    if (given(bias)) {
        FL_VALUE(bias->dim() == 1 && bias->size(0) == n, "linear: bias must be [", n, "], got ", shape_text(bias->sizes()));
        FL_VALUE(bias->scalar_type() == x.scalar_type(), "linear: tensors of one dtype, got ", x.scalar_type(), " and ",
                 bias->scalar_type());
    }
    no_tangent("linear", {x, w, bias, residual});
    const bool flat = x.dim() == 2;
    std::vector<int64_t> shape;
    if (!flat || given(residual)) {
        shape = x.sizes().vec();
        shape.back() = n;
    }
    if (given(residual)) {
        FL_VALUE(residual->sizes() == at::IntArrayRef(shape), "linear: residual must be ", shape_text(shape), ", got ",
                 shape_text(residual->sizes()));
        FL_VALUE(residual->scalar_type() == x.scalar_type(), "linear: tensors of one dtype, got ", x.scalar_type(), " and ",
                 residual->scalar_type());
    }
    const Tensor x2 = flat ? x : x.reshape({-1, k});
    const OptTensor res2 = given(residual) && !flat ? OptTensor(residual->reshape({-1, n})) : residual;
    Tensor y;
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(bias) || wants_grad(residual)))
        y = Linear::apply(x2, w, bias, res2, act);
    else
        y = std::get<0>(linear_forward(x2, w, bias, res2, act, false, std::nullopt));
    return flat ? y : y.view(shape);
}

// ---- the hops' weights ------------------------------------------------------------
struct Rules {
    double tau, repetition, frequency, presence;
};

fl_weights weights_params(const Tensor &z, const OptTensor &bias, const OptTensor &mask, const OptTensor &states,
                          const OptTensor &history, const Rules &r) {
    fl_weights p{};
    p.logits = ptr(z);
    p.bias = ptr(bias);
    p.mask = ptr(mask);
    p.states = ptr<int64_t>(states);
    p.history = ptr<int64_t>(history);
    p.ld = ld(z);
    p.rows = z.size(0);
    p.n = z.size(1);
    p.bias_ld = given(bias) && bias->dim() == 2 ? p.n : 0;
    if (given(mask)) {
        p.mask_ld = ld(*mask);
        p.n_states = mask->size(0);
    }
    if (given(history)) {
        p.hist_ld = ld(*history);
        p.hist = history->size(1);
    }
    p.tau = r.tau;
    p.repetition = r.repetition;
    p.frequency = r.frequency;
    p.presence = r.presence;
    p.dtype = dtype_of(z);
    return p;
}

// On 2-D tensors the library can address (unit inner strides).
Tensor weights_forward(const Tensor &z, const OptTensor &bias, const OptTensor &mask, const OptTensor &states,
                       const OptTensor &history, double tau, double repetition, double frequency, double presence,
                       const OptTensor &out) {
    Devices d{"relation weights"};
    d.add(z);
    d.add(bias);
    d.add(mask);
    d.add(states);
    d.add(history);
    d.add(out);
    Tensor w = given(out) ? *out : at::empty(z.sizes(), z.options().dtype(at::kFloat));
    if (w.numel() == 0) return w;
    const fl_weights p = weights_params(z, bias, mask, states, history, {tau, repetition, frequency, presence});
    OnDevice on(z);
    check(fl_relation_weights(&p, ptr<float>(w), on.stream), "relation weights");
    if (given(out)) written(w);
    return w;
}

std::tuple<Tensor, Tensor> weights_backward(const Tensor &w, const Tensor &g0, const Tensor &z, const OptTensor &bias,
                                            const OptTensor &history, double tau, double repetition, bool want_logits,
                                            bool want_bias) {
    Devices d{"relation weights backward"};
    d.add(w);
    d.add(g0);
    d.add(z);
    d.add(bias);
    d.add(history);
    const Tensor g = g0.stride(1) == 1 ? g0 : g0.contiguous();
    Tensor dz = want_logits ? at::empty(w.sizes(), z.options()) : Tensor();
    Tensor db = want_bias ? at::empty(bias->sizes(), bias->options()) : Tensor();
    const fl_weights p = weights_params(z, bias, std::nullopt, std::nullopt, history, {tau, repetition, 0.0, 0.0});
    OnDevice on(w);
    const size_t bytes = want_bias && bias->dim() == 1 ? fl_relation_weights_workspace(w.size(0), w.size(1)) : 0;
    const Tensor ws = workspace(bytes, w);
    check(fl_relation_weights_backward(&p, ptr<float>(w), ptr<float>(g), g.stride(0), ptr(dz), ptr(db), ptr(ws), bytes,
                                       on.stream),
          "relation weights backward");
    return {dz, db};
}

struct Weights : torch::autograd::Function<Weights> {
    static Tensor forward(AutogradContext *ctx, const Tensor &z, const OptTensor &bias, const OptTensor &mask,
                          const OptTensor &states, const OptTensor &history, double tau, double repetition,
                          double frequency, double presence) {
        Tensor w = weights_forward(z, bias, mask, states, history, tau, repetition, frequency, presence, std::nullopt);
        ctx->saved_data["tau"] = tau;
        ctx->saved_data["repetition"] = repetition;
        ctx->saved_data["bias"] = given(bias);
        // the history matters to the gradient through the sign of penalised logits only
        ctx->save_for_backward({w, z, given(bias) ? *bias : Tensor(),
                                given(history) && repetition != 1.0 ? *history : Tensor()});
        return w;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(9);
        const Tensor g = grads[0];
        if (!g.defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const Tensor &w = saved[0], &z = saved[1];
        const bool want_z = ctx->needs_input_grad(0);
        const bool want_bias = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(1);
        if (w.numel() == 0) {
            if (want_z) out[0] = at::zeros_like(z);
            if (want_bias) out[1] = at::zeros_like(saved[2]);
            return out;
        }
        Tensor dz, db;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            std::tie(dz, db) = weights_backward(w, g, z, saved[2], saved[3], ctx->saved_data["tau"].toDouble(),
                                                ctx->saved_data["repetition"].toDouble(), want_z, want_bias);
        }
        // both are made of the weights, which logits and bias have a part in
        out[0] = once(dz, g, z, saved[2]);
        out[1] = once(db, g, z, saved[2]);
        return out;
    }
};

Tensor relation_weights(const Tensor &logits, double tau, const OptTensor &mask0, const OptTensor &states0,
                        const OptTensor &bias0, const OptTensor &history0, double repetition, double frequency,
                        double presence) {
    FL_VALUE(logits.dim() >= 1 && dtype_of(logits) >= 0,
             "relation_weights takes float32, float16 or bfloat16 logits [..., n], got ", logits.scalar_type());
    const int64_t n = logits.size(-1);
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    FL_VALUE(n >= 1 && n <= kMaxColumns, "relation_weights: need 1 to ", kMaxColumns, " operators, got ", n);
    // compared as the fp32 values that the kernels use
    FL_VALUE(tau > 1e-30 && tau < 1e30 && repetition > 1e-30 && repetition < 1e30,
             "relation_weights: tau and repetition must be positive, got ", tau, " and ", repetition);
    FL_VALUE(std::fabs(frequency) < 1e30 && std::fabs(presence) < 1e30,
             "relation_weights: penalties must be finite, got ", frequency, " and ", presence);
    auto is_row = [&](const Tensor &t) { return t.dim() == 1 && t.size(0) == n; };
    if (given(bias0))
        FL_VALUE(bias0->scalar_type() == logits.scalar_type() && (is_row(*bias0) || bias0->sizes() == logits.sizes()),
                 "relation_weights: bias must be [", n, "] or the logits' shape, of their dtype");
    if (given(mask0)) {
        FL_VALUE(mask0->scalar_type() == at::kBool || mask0->scalar_type() == at::kByte,
                 "relation_weights: mask must be bool or uint8, got ", mask0->scalar_type());
        const bool ok = given(states0) ? mask0->dim() == 2 && mask0->size(1) == n && mask0->size(0) > 0
                                       : is_row(*mask0) || mask0->sizes() == logits.sizes();
        FL_VALUE(ok, "relation_weights: mask must be [states, ", n, "] with states, else [", n,
                 "] or the logits' shape, got ", shape_text(mask0->sizes()));
    }
    if (given(states0))
        FL_VALUE(given(mask0) && states0->scalar_type() == at::kLong && states0->sizes() == lead,
                 "relation_weights: states must be int64 ", shape_text(lead), ", next to a mask");
    if (given(history0)) {
        FL_VALUE(history0->scalar_type() == at::kLong && history0->dim() >= 1 &&
                     history0->sizes().slice(0, history0->dim() - 1) == lead,
                 "relation_weights: history must be int64 ", shape_text(lead), " + [H]");
        FL_VALUE(history0->size(-1) <= kMaxHistory, "relation_weights: at most ", kMaxHistory, " history entries, got ",
                 history0->size(-1));
    }
    no_tangent("relation_weights", {logits, bias0});
    const bool flat = logits.dim() == 2;
    const Tensor z = lines(flat ? logits : logits.reshape({-1, n}));
    OptTensor bias, mask, states, history;
    if (given(bias0)) bias = bias0->dim() == 1 ? bias0->contiguous() : bias0->reshape({-1, n}).contiguous();
    if (given(mask0)) mask = lines(mask0->dim() == 2 ? *mask0 : mask0->reshape({-1, n}));
    if (given(states0)) states = (states0->dim() == 1 ? *states0 : states0->reshape({-1})).contiguous();
    if (given(history0) && history0->size(-1) > 0)
        history = lines(history0->dim() == 2 ? *history0 : history0->reshape({-1, history0->size(-1)}));
    Tensor w;
    if (at::GradMode::is_enabled() && (wants_grad(z) || wants_grad(bias)))
        w = Weights::apply(z, bias, mask, states, history, tau, repetition, frequency, presence);
    else
        w = weights_forward(z, bias, mask, states, history, tau, repetition, frequency, presence, std::nullopt);
    return flat ? w : w.view(logits.sizes());
}

// ---- orthogonalised updates ---------------------------------------------------------
using Coefficients = std::tuple<double, double, double>;

// A common (b1, b2) of tensors [..., m, n] of one shape, with each one's strides; false when the leading
// dimensions of some need more than two strides.
bool as_batch(at::ArrayRef<Tensor> ts, int64_t &b1, int64_t &b2, std::vector<fl_matrices> &out) {
    const auto sizes = ts[0].sizes();
    int64_t total = 1;
    const int64_t leading = ts[0].dim() - 2;
    for (int64_t i = 0; i < leading; ++i) total *= sizes[i];
    struct Dim {
        int64_t n, s;
    };
    std::vector<std::vector<Dim>> merged;
    int64_t split = 1;  // b2, the innermost batch dimensions that every tensor holds at one stride
    for (const Tensor &t : ts) {
        std::vector<Dim> dims;
        for (int64_t i = 0; i < leading; ++i) {
            const int64_t n = sizes[i], s = t.stride(i);
            if (n == 1) continue;
            if (!dims.empty() && dims.back().s == n * s) dims.back() = Dim{dims.back().n * n, s};
            else dims.push_back(Dim{n, s});
        }
        if (dims.size() > 2 || (dims.size() == 2 && split != 1 && split != dims[1].n)) return false;
        if (dims.size() == 2) split = dims[1].n;
        merged.push_back(std::move(dims));
    }
    out.clear();
    for (size_t i = 0; i < ts.size(); ++i) {
        const auto &dims = merged[i];
        fl_matrices f{};
        f.ptr = ptr(ts[i]);
        f.stride_b2 = dims.empty() ? 0 : dims.back().s;
        f.stride_b1 = dims.size() == 2 ? dims[0].s : f.stride_b2 * split;
        f.stride_i = ts[i].stride(-2);
        f.stride_j = ts[i].stride(-1);
        out.push_back(f);
    }
    b1 = total / split;
    b2 = split;
    return true;
}

Tensor orthogonalize(const Tensor &update, int64_t steps, const Coefficients &c, double eps) {
    Devices d{"orthogonalize"};
    d.add(update);
    no_tangent("orthogonalize", {update});
    Tensor out = at::empty(update.sizes(), update.options());
    if (out.numel() == 0) return out;
    int64_t b1, b2;
    std::vector<fl_matrices> f;
    Tensor u = update;
    if (!as_batch({u, out}, b1, b2, f)) {  // strides that two batch dimensions cannot express
        u = update.contiguous();
        as_batch({u, out}, b1, b2, f);
    }
    const int64_t m = update.size(-2), n = update.size(-1);
    OnDevice on(update);
    const size_t bytes = fl_newton_schulz_workspace(b1 * b2, m, n, static_cast<int>(steps));
    const Tensor ws = workspace(bytes, update);
    check(fl_orthogonalize(&f[0], &f[1], b1, b2, m, n, dtype_of(update), static_cast<int>(steps), std::get<0>(c),
                           std::get<1>(c), std::get<2>(c), eps, ptr(ws), bytes, on.stream),
          "orthogonalize");
    return out;
}

void muon_update(const Tensor &param, const Tensor &grad, const Tensor &momentum, const Tensor &param_out,
                 const Tensor &momentum_out, double lr, double beta, bool nesterov, double weight_decay, double scale,
                 int64_t steps, const Coefficients &c, double eps, const OptTensor &gate) {
    Devices d{"muon_update"};
    d.add(param);
    d.add(grad);
    d.add(momentum);
    d.add(param_out);
    d.add(momentum_out);
    d.add(gate);
    no_tangent("muon_update", {param, grad, momentum});
    if (param.numel() == 0) return;
    int64_t b1, b2;
    std::vector<fl_matrices> f;
    if (!as_batch({param, grad, momentum, param_out, momentum_out}, b1, b2, f)) {
        // strides that two batch dimensions cannot express: through plain copies
        Tensor p = at::empty(param.sizes(), param.options()), m = at::empty(param.sizes(), param.options());
        muon_update(param.contiguous(), grad.contiguous(), momentum.contiguous(), p, m, lr, beta, nesterov, weight_decay,
                    scale, steps, c, eps, gate);
        param_out.copy_(p);
        momentum_out.copy_(m);
        return;
    }
    const int64_t m = param.size(-2), n = param.size(-1);
    OnDevice on(param);
    const size_t bytes = fl_newton_schulz_workspace(b1 * b2, m, n, static_cast<int>(steps));
    const Tensor ws = workspace(bytes, param);
    check(fl_muon_update(&f[0], &f[1], &f[2], &f[3], &f[4], b1, b2, m, n, lr, beta, nesterov, weight_decay, scale,
                         static_cast<int>(steps), std::get<0>(c), std::get<1>(c), std::get<2>(c), eps, ptr<float>(gate),
                         ptr(ws), bytes, on.stream),
          "muon_update");
    written(param_out);
    written(momentum_out);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    m.def("linear", &linear);
    m.def("linear_forward", &linear_forward);
    m.def("linear_backward", &linear_backward);
    m.def("relation_weights", &relation_weights);
    m.def("weights_forward", &weights_forward);
    m.def("weights_backward", &weights_backward);
    m.def("orthogonalize", &orthogonalize);
    m.def("muon_update", &muon_update);
}
