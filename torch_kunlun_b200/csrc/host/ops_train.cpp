// ops_train.cpp -- the training operators of the kunlun backend that have no
// aten name: dropout with a recomputed mask, the residual norm and the linear
// cross entropy, each an autograd function over one or two calls of the C ABI.
//
// The reference stops at linear, convolution, relu and MSE gradients
// (csrc/autograd.cpp) and at a forward layer_norm (csrc/ops_nn.cpp:85-130);
// these ops follow its float16/float32 rules.  Their backward passes are not
// differentiable themselves and say so.
#include <ATen/EmptyTensor.h>
#include <torch/csrc/autograd/custom_function.h>

#include "kunlun.h"

namespace torch_kunlun {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct DeviceScope {
    int prev;
    explicit DeviceScope(int dev) : prev(current_device()) {
        if (dev >= 0 && dev != prev) cudaSetDevice(dev);
    }
    ~DeviceScope() { cudaSetDevice(prev); }
};

// An autograd function takes an absent tensor as an empty optional.
using Optional = std::optional<at::Tensor>;
Optional optional(const at::Tensor& t) { return t.defined() ? Optional(t) : Optional(); }
at::Tensor or_undefined(const Optional& t) { return t.has_value() ? *t : at::Tensor(); }

void check_input(const at::Tensor& t, const char* op) {
    TORCH_CHECK(t.defined() && t.device().type() == c10::DeviceType::PrivateUse1, "kunlun ", op,
                " requires kunlun tensors, got ", t.device());
    TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat, "kunlun ", op,
                " supports float16/float32, got ", t.scalar_type());
}

// A parameter of x's dtype on x's device, contiguous; undefined when absent.
at::Tensor param(const std::optional<at::Tensor>& t, const at::Tensor& x, const char* op, const char* name) {
    if (!t.has_value() || !t->defined()) return at::Tensor();
    TORCH_CHECK(t->device() == x.device(), "kunlun ", op, ": ", name, " is on ", t->device(), ", expected ", x.device());
    TORCH_CHECK(t->scalar_type() == x.scalar_type(), "kunlun ", op, ": ", name, " must be ", x.scalar_type(), ", got ",
                t->scalar_type());
    return t->contiguous();
}

bool needs_grad(std::initializer_list<at::Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// A dual tensor would come back without its tangent where no gradient is wanted.
void check_no_tangent(const char* op, std::initializer_list<at::Tensor> ts) {
    for (const at::Tensor& t : ts)
        TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "kunlun ", op, ": forward-mode derivatives are not implemented");
}

void check_single_backward(const char* op) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "kunlun ", op, ": gradients of its backward pass (create_graph=True) are not implemented");
}

// A saved tensor as the kernels take it.  Saved-tensor hooks may hand back other
// tensors than were saved, so what the pointers rest on is looked at again.
at::Tensor restored(const at::Tensor& t, at::Device device, at::ScalarType type, at::IntArrayRef sizes, const char* op, const char* name) {
    TORCH_CHECK(t.defined() && t.device() == device && t.scalar_type() == type && t.sizes().equals(sizes), "kunlun ", op, ": the saved ", name,
                " came back as ", t.defined() ? t.toString() : "nothing", " ", t.defined() ? t.sizes() : at::IntArrayRef(), " on ",
                t.defined() ? t.device() : at::Device(at::kCPU), ", expected ", type, " ", sizes, " on ", device);
    return t.contiguous();
}

// The tensor inputs, of those in `given`, whose gradients this backward pass has
// been asked for (an input that requires none, or that autograd.grad leaves out,
// is not).
unsigned wanted_gradients(AutogradContext* ctx, unsigned given) {
    unsigned wanted = 0;
    for (size_t i = 0, edge = 0; given >> i != 0; ++i)
        if (given >> i & 1u) wanted |= (ctx->needs_input_grad(edge++) ? 1u : 0u) << i;
    return wanted;
}

// A contiguous tensor on the current device, allocated without a trip through
// the dispatcher: these ops allocate up to nine tensors a call.
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type) {
    return at::detail::empty_generic(shape, get_allocator(), c10::DispatchKeySet(c10::DispatchKey::PrivateUse1), type,
                                     std::nullopt);
}

at::Tensor scratch(size_t bytes) { return fresh({static_cast<int64_t>(bytes + 1024)}, at::kByte); }

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- dropout --------------------------------------------------------------------

at::Tensor dropout_run(const at::Tensor& x, double p, uint64_t seed, uint64_t offset) {
    at::Tensor xc = x.contiguous();
    const int dev = xc.device().index();
    DeviceScope g(dev);
    at::Tensor y = fresh(xc.sizes(), xc.scalar_type());
    check_tk(tk_dropout(tk_dtype(xc.scalar_type()), ptr(xc), ptr(y), xc.numel(), p, seed, offset, current_stream(dev)),
             "tk_dropout");
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, double p, int64_t seed, int64_t offset) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        return dropout_run(x, p, static_cast<uint64_t>(seed), static_cast<uint64_t>(offset));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_single_backward("dropout");
        at::Tensor gx = dropout_run(grads[0], ctx->saved_data["p"].toDouble(),
                                    static_cast<uint64_t>(ctx->saved_data["seed"].toInt()),
                                    static_cast<uint64_t>(ctx->saved_data["offset"].toInt()));
        return {gx, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// ---- residual norm ----------------------------------------------------------------

struct NormOptions {
    bool rms, post;
    double scale, eps, p;
    int64_t seed, offset;
};

tk_residual_norm_desc_t norm_desc(const at::Tensor& like, const NormOptions& o, const at::Tensor& weight,
                                  const at::Tensor& post_weight, const at::Tensor& post_bias, const at::Tensor& gate) {
    tk_residual_norm_desc_t d = {};
    d.dtype = tk_dtype(like.scalar_type());
    d.norm = o.rms ? TK_NORM_RMS : TK_NORM_LAYER;
    d.cols = like.size(-1);
    d.rows = like.numel() / d.cols;
    d.weight = ptr(weight);
    d.post_norm = o.post ? 1 : 0;
    d.post_weight = ptr(post_weight);
    d.post_bias = ptr(post_bias);
    d.gate = ptr(gate);
    d.gate_rows = gate.defined() ? gate.numel() / d.cols : 0;
    d.residual_scale = static_cast<float>(o.scale);
    d.eps = static_cast<float>(o.eps);
    d.p = o.p;
    d.seed = static_cast<uint64_t>(o.seed);
    d.offset = static_cast<uint64_t>(o.offset);
    return d;
}

std::tuple<at::Tensor, at::Tensor> norm_run(const at::Tensor& x, const at::Tensor& f, const at::Tensor& weight,
                                            const at::Tensor& bias, const at::Tensor& post_weight,
                                            const at::Tensor& post_bias, const at::Tensor& gate, const NormOptions& o,
                                            const at::Tensor& stats) {
    const int dev = x.device().index();
    DeviceScope g(dev);
    at::Tensor x_new = fresh(x.sizes(), x.scalar_type()), h = fresh(x.sizes(), x.scalar_type());
    tk_residual_norm_desc_t d = norm_desc(x, o, weight, post_weight, post_bias, gate);
    d.x = ptr(x);
    d.f = ptr(f);
    d.bias = ptr(bias);
    d.x_new = ptr(x_new);
    d.h = ptr(h);
    d.stats = stats.defined() ? stats.data_ptr<float>() : nullptr;
    check_tk(tk_residual_norm(&d, current_stream(dev)), "tk_residual_norm");
    return {x_new, h};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& f, const Optional& weight_in,
                                 const Optional& bias_in, const Optional& post_weight_in, const Optional& post_bias_in,
                                 const Optional& gate_in, const NormOptions& o) {
        const at::Tensor weight = or_undefined(weight_in), bias = or_undefined(bias_in),
                         post_weight = or_undefined(post_weight_in), post_bias = or_undefined(post_bias_in),
                         gate = or_undefined(gate_in);
        const int64_t rows = x.numel() / x.size(-1);
        at::Tensor stats;
        {
            DeviceScope g(x.device().index());
            stats = fresh({rows, 4}, at::kFloat);
        }
        auto [x_new, h] = norm_run(x, f, weight, bias, post_weight, post_bias, gate, o, stats);
        ctx->save_for_backward({x, f, weight, post_weight, post_bias, gate, stats});
        int64_t given = 0;  // a bit for each tensor
        const at::Tensor* const inputs[7] = {&x, &f, &weight, &bias, &post_weight, &post_bias, &gate};
        for (int i = 0; i < 7; ++i)
            if (inputs[i]->defined()) given |= 1 << i;
        std::vector<int64_t> ints = {o.rms, o.post, o.seed, o.offset, given, static_cast<int64_t>(x.scalar_type()), x.device().index(), x.dim()};
        ints.insert(ints.end(), x.sizes().begin(), x.sizes().end());
        if (gate.defined()) ints.insert(ints.end(), gate.sizes().begin(), gate.sizes().end());
        ctx->saved_data["ints"] = std::move(ints);
        ctx->saved_data["reals"] = std::vector<double>{o.scale, o.eps, o.p};
        ctx->set_materialize_grads(false);
        return {x_new, h};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_single_backward("residual_norm");
        variable_list out(8);
        at::Tensor gx = grads[0], gh = grads[1];
        if (!gx.defined() && !gh.defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const auto ints = ctx->saved_data["ints"].toIntVector();
        const auto real = ctx->saved_data["reals"].toDoubleVector();
        const NormOptions o = {ints[0] != 0, ints[1] != 0, real[0], real[1], real[2], ints[2], ints[3]};
        const auto given = [&](int i) { return (ints[4] >> i & 1) != 0; };
        const unsigned wanted = wanted_gradients(ctx, static_cast<unsigned>(ints[4]));
        if (wanted == 0) return out;
        const at::ScalarType type = static_cast<at::ScalarType>(ints[5]);
        const at::Device device(c10::DeviceType::PrivateUse1, static_cast<at::DeviceIndex>(ints[6]));
        const at::IntArrayRef shapes = at::IntArrayRef(ints).slice(8), sizes = shapes.slice(0, ints[7]), gate_sizes = shapes.slice(ints[7]);
        const int64_t cols = sizes.back(), rows = c10::multiply_integers(sizes) / cols;
        const auto again = [&](int i, const char* name, at::IntArrayRef shape) { return restored(saved[i], device, type, shape, "residual_norm", name); };
        const at::Tensor x = again(0, "x", sizes), f = again(1, "f", sizes),
                         weight = given(2) ? again(2, "weight", cols) : at::Tensor(),
                         post_weight = given(4) ? again(3, "post_weight", cols) : at::Tensor(),
                         post_bias = given(5) ? again(4, "post_bias", cols) : at::Tensor(),
                         gate = given(6) ? again(5, "gate", gate_sizes) : at::Tensor(),
                         stats = restored(saved[6], device, at::kFloat, {rows, 4}, "residual_norm", "statistics");
        if (gx.defined()) gx = gx.contiguous();
        if (gh.defined()) gh = gh.contiguous();
        const int dev = device.index();
        DeviceScope g(dev);
        if (wanted >> 0 & 1) out[0] = fresh(x.sizes(), type);
        if (wanted >> 1 & 1) out[1] = fresh(x.sizes(), type);
        if (wanted >> 2 & 1) out[2] = fresh({cols}, type);
        if (wanted >> 3 & 1) out[3] = fresh({cols}, type);
        if (wanted >> 4 & 1) out[4] = fresh({cols}, type);
        if (wanted >> 5 & 1) out[5] = fresh({cols}, type);
        if (wanted >> 6 & 1) out[6] = fresh(gate.sizes(), type);
        tk_residual_norm_grad_desc_t d = {};
        d.fwd = norm_desc(x, o, weight, post_weight, post_bias, gate);
        d.fwd.x = ptr(x);
        d.fwd.f = ptr(f);
        d.fwd.stats = stats.data_ptr<float>();
        d.grad_x_new = ptr(gx);
        d.grad_h = ptr(gh);
        d.dx = ptr(out[0]);
        d.df = ptr(out[1]);
        d.dweight = ptr(out[2]);
        d.dbias = ptr(out[3]);
        d.dpost_weight = ptr(out[4]);
        d.dpost_bias = ptr(out[5]);
        d.dgate = ptr(out[6]);
        const size_t bytes = tk_residual_norm_backward_workspace_size(&d);
        TORCH_CHECK(bytes > 0, "kunlun residual_norm: ", tk_last_error_string());
        at::Tensor ws = scratch(bytes);
        check_tk(tk_residual_norm_backward(&d, aligned_base(ws), bytes, current_stream(dev)), "tk_residual_norm_backward");
        return out;
    }
};

// ---- linear cross entropy ------------------------------------------------------------

tk_linear_ce_desc_t ce_desc(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& target, const at::Tensor& bias,
                            int64_t ignore_index, int64_t reduction) {
    tk_linear_ce_desc_t d = {};
    d.dtype = tk_dtype(weight.scalar_type());
    d.rows = target.size(0);
    d.cols = weight.size(1);
    d.vocab = weight.size(0);
    d.x = ptr(x);
    d.weight = ptr(weight);
    d.bias = ptr(bias);
    d.target = target.numel() > 0 ? target.data_ptr<int64_t>() : nullptr;
    d.ignore_index = ignore_index;
    d.reduction = static_cast<int>(reduction);
    return d;
}

// x [N, D], weight [V, D], target [N]; `state` (when defined) is filled for
// the backward pass.
at::Tensor ce_run(tk_linear_ce_desc_t d, const at::Tensor& x, at::Tensor* state) {
    const int dev = x.device().index();
    DeviceScope g(dev);
    at::Tensor loss = d.reduction == TK_REDUCE_NONE ? fresh({d.rows}, at::kFloat) : fresh({}, at::kFloat);
    d.loss = d.reduction == TK_REDUCE_NONE && d.rows == 0 ? nullptr : loss.data_ptr<float>();
    const size_t bytes = tk_linear_ce_workspace_size(&d);
    TORCH_CHECK(bytes > 0, "kunlun linear_cross_entropy: ", tk_last_error_string());
    if (state != nullptr) {
        *state = fresh({static_cast<int64_t>(tk_linear_ce_state_size(&d))}, at::kByte);
        d.state = state->data_ptr();
    }
    at::Tensor ws = scratch(bytes);
    check_tk(tk_linear_ce(&d, aligned_base(ws), bytes, current_stream(dev)), "tk_linear_ce");
    return loss;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& target,
                              const Optional& bias_in, int64_t ignore_index, int64_t reduction) {
        const at::Tensor bias = or_undefined(bias_in);
        at::Tensor state;
        at::Tensor loss = ce_run(ce_desc(x, weight, target, bias, ignore_index, reduction), x, &state);
        ctx->save_for_backward({weight, target, bias, state});  // the state holds x's rows
        ctx->saved_data["ints"] = std::vector<int64_t>{ignore_index, reduction, bias.defined(), x.size(0), x.size(1), weight.size(0), state.numel(),
                                                       static_cast<int64_t>(x.scalar_type()), x.device().index()};
        ctx->set_materialize_grads(false);
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_single_backward("linear_cross_entropy");
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const auto ints = ctx->saved_data["ints"].toIntVector();
        const unsigned wanted = wanted_gradients(ctx, ints[2] ? 0b1111u : 0b111u);  // x, weight, target, bias
        if (wanted == 0) return out;
        const int64_t rows = ints[3], cols = ints[4], vocab = ints[5];
        const at::ScalarType type = static_cast<at::ScalarType>(ints[7]);
        const at::Device device(c10::DeviceType::PrivateUse1, static_cast<at::DeviceIndex>(ints[8]));
        const auto again = [&](int i, const char* name, at::ScalarType t, at::IntArrayRef shape) {
            return restored(saved[i], device, t, shape, "linear_cross_entropy", name);
        };
        const at::Tensor weight = again(0, "weight", type, {vocab, cols}), target = again(1, "target", at::kLong, rows),
                         bias = ints[2] ? again(2, "bias", type, vocab) : at::Tensor(), state = again(3, "state", at::kByte, ints[6]);
        const int dev = device.index();
        DeviceScope g(dev);
        const at::Tensor grad = grads[0].contiguous();
        if (wanted & 1u) out[0] = fresh({rows, cols}, type);
        if (wanted & 2u) out[1] = fresh(weight.sizes(), type);
        if (wanted & 8u) out[3] = fresh(bias.sizes(), type);
        tk_linear_ce_grad_desc_t d = {};
        d.fwd = ce_desc(at::Tensor(), weight, target, bias, ints[0], ints[1]);
        d.fwd.state = state.data_ptr();
        d.grad_loss = grad.numel() > 0 ? grad.data_ptr<float>() : nullptr;
        d.dx = ptr(out[0]);
        d.dweight = ptr(out[1]);
        d.dbias = ptr(out[3]);
        const size_t bytes = tk_linear_ce_backward_workspace_size(&d);
        TORCH_CHECK(bytes > 0, "kunlun linear_cross_entropy: ", tk_last_error_string());
        at::Tensor ws = scratch(bytes);
        check_tk(tk_linear_ce_backward(&d, aligned_base(ws), bytes, current_stream(dev)), "tk_linear_ce_backward");
        return out;
    }
};

}  // namespace

at::Tensor linear_cross_entropy(const at::Tensor& x_in, const at::Tensor& weight_in, const at::Tensor& target_in,
                                const std::optional<at::Tensor>& bias_in, int64_t ignore_index, int64_t reduction) {
    const char* op = "linear_cross_entropy";
    check_input(x_in, op);
    TORCH_CHECK(x_in.dim() >= 1 && x_in.size(-1) >= 1, "kunlun linear_cross_entropy: x needs a last dimension of at least 1");
    TORCH_CHECK(weight_in.defined() && weight_in.dim() == 2 && weight_in.size(0) >= 1 && weight_in.size(1) == x_in.size(-1),
                "kunlun linear_cross_entropy: weight must be [vocab, ", x_in.size(-1), "], got ", weight_in.sizes());
    TORCH_CHECK(target_in.device() == x_in.device() && target_in.scalar_type() == at::kLong,
                "kunlun linear_cross_entropy: target must be int64 on ", x_in.device(), ", got ", target_in.scalar_type(),
                " on ", target_in.device());
    TORCH_CHECK(target_in.sizes().equals(x_in.sizes().slice(0, x_in.dim() - 1)),
                "kunlun linear_cross_entropy: target has shape ", target_in.sizes(), ", expected x's leading dimensions of ",
                x_in.sizes());
    TORCH_CHECK(reduction >= 0 && reduction <= 2, "kunlun linear_cross_entropy: bad reduction ", reduction);
    const at::Tensor weight = param(weight_in, x_in, op, "weight"), bias = param(bias_in, x_in, op, "bias");
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == weight.size(0)),
                "kunlun linear_cross_entropy: bias must be [", weight.size(0), "], got ", bias.sizes());
    check_no_tangent(op, {x_in, weight, bias});
    const int64_t cols = x_in.size(-1), rows = x_in.numel() / cols;
    const at::Tensor x = x_in.contiguous().view({rows, cols}), target = target_in.contiguous().view({rows});
    at::Tensor loss;
    if (needs_grad({x, weight, bias})) {
        loss = LinearCrossEntropy::apply(x, weight, target, optional(bias), ignore_index, reduction);
    } else {
        at::AutoDispatchBelowADInplaceOrView guard;
        loss = ce_run(ce_desc(x, weight, target, bias, ignore_index, reduction), x, nullptr);
    }
    return reduction == TK_REDUCE_NONE ? loss.view(target_in.sizes()) : loss;
}

at::Tensor dropout(const at::Tensor& x, double p, uint64_t seed, uint64_t offset) {
    check_input(x, "dropout");
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "kunlun dropout: p must be in [0, 1], got ", p);
    check_no_tangent("dropout", {x});
    if (needs_grad({x})) return Dropout::apply(x, p, static_cast<int64_t>(seed), static_cast<int64_t>(offset));
    at::AutoDispatchBelowADInplaceOrView guard;
    return dropout_run(x, p, seed, offset);
}

std::tuple<at::Tensor, at::Tensor> residual_norm(
    const at::Tensor& x_in, const at::Tensor& f_in, const std::optional<at::Tensor>& weight_in,
    const std::optional<at::Tensor>& bias_in, bool rms, bool post_norm, const std::optional<at::Tensor>& post_weight_in,
    const std::optional<at::Tensor>& post_bias_in, const std::optional<at::Tensor>& gate_in, double residual_scale,
    double eps, double p, uint64_t seed, uint64_t offset) {
    const char* op = "residual_norm";
    check_input(x_in, op);
    check_input(f_in, op);
    TORCH_CHECK(x_in.dim() >= 1 && x_in.size(-1) >= 1, "kunlun residual_norm: x needs a last dimension of at least 1");
    TORCH_CHECK(f_in.sizes().equals(x_in.sizes()), "kunlun residual_norm: f has shape ", f_in.sizes(), ", expected ", x_in.sizes());
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "kunlun residual_norm: p must be in [0, 1], got ", p);
    TORCH_CHECK(post_norm || !((post_weight_in.has_value() && post_weight_in->defined()) ||
                               (post_bias_in.has_value() && post_bias_in->defined())),
                "kunlun residual_norm: post_weight and post_bias need post_norm=True");
    const at::Tensor f = param(f_in, x_in, op, "f"), weight = param(weight_in, x_in, op, "weight"),
                     bias = param(bias_in, x_in, op, "bias"), post_weight = param(post_weight_in, x_in, op, "post_weight"),
                     post_bias = param(post_bias_in, x_in, op, "post_bias"), gate = param(gate_in, x_in, op, "gate"),
                     x = x_in.contiguous();
    const int64_t cols = x.size(-1);
    for (const at::Tensor& t : {weight, bias, post_weight, post_bias})
        TORCH_CHECK(!t.defined() || (t.dim() == 1 && t.size(0) == cols), "kunlun residual_norm: weights and biases must be [",
                    cols, "], got ", t.sizes());
    if (gate.defined() && !(gate.dim() == 1 && gate.size(0) == cols)) {
        bool ok = gate.dim() == x.dim() && gate.size(-1) == cols, shared = false;
        for (int64_t i = 0; ok && i + 1 < x.dim(); ++i) {
            if (gate.size(i) != x.size(i)) shared = true;
            ok = shared ? gate.size(i) == 1 : true;
        }
        TORCH_CHECK(ok, "kunlun residual_norm: gate must be [", cols, "] or x's shape ", x.sizes(),
                    " with 1 in place of some last dimensions before the columns, got ", gate.sizes());
    }
    check_no_tangent(op, {x, f, weight, bias, post_weight, post_bias, gate});
    const NormOptions o = {rms, post_norm, residual_scale, eps, p, static_cast<int64_t>(seed), static_cast<int64_t>(offset)};
    if (needs_grad({x, f, weight, bias, post_weight, post_bias, gate})) {
        const variable_list r = ResidualNorm::apply(x, f, optional(weight), optional(bias), optional(post_weight),
                                                    optional(post_bias), optional(gate), o);
        return {r[0], r[1]};
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    return norm_run(x, f, weight, bias, post_weight, post_bias, gate, o, at::Tensor());
}

}  // namespace torch_kunlun
