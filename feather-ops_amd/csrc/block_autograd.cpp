// The gradients of rms_norm and silu_mul as nodes of torch's autograd graph, in C++. The backward of a CUDA tensor runs on a
// thread of its own, and a Python function there has to take the interpreter's lock and pull its data to another core: with
// Python nodes the norm's forward and backward at 4 x 256 took 112 us where one thread took 51 (gate 65 and 29, a product
// with a number, a node of torch's own, 51 and 23), whatever its kernels took; with these the norm 87, the gate 50. Host code; unlike the ops themselves
// (block_extension.cpp) it needs torch's C++ interface and not only its stable one, and is a library of its own for that.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

template <typename Signature>
c10::TypedOperatorHandle<Signature> op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

Tensor silu_mul(const Tensor& x) {
    static const auto call = op<Tensor(const Tensor&)>("feather_ops::silu_mul");
    return call.call(x);
}

Tensor silu_mul_backward(const Tensor& grad_y, const Tensor& x) {
    static const auto call = op<Tensor(const Tensor&, const Tensor&)>("feather_ops::silu_mul_backward");
    return call.call(grad_y, x);
}

using Norm = std::tuple<Tensor, Tensor, Tensor>;

Norm rms_norm(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual, double eps, bool need_rstd) {
    static const auto call =
        op<Norm(const Tensor&, const Tensor&, const std::optional<Tensor>&, double, bool)>("feather_ops::rms_norm");
    return call.call(x, weight, residual, eps, need_rstd);
}

std::tuple<Tensor, Tensor> rms_norm_backward(const Tensor& grad_y, const std::optional<Tensor>& grad_h, const Tensor& h,
                                             const Tensor& weight, const Tensor& rstd, bool need_weight) {
    static const auto call =
        op<std::tuple<Tensor, Tensor>(const Tensor&, const std::optional<Tensor>&, const Tensor&, const Tensor&,
                                      const Tensor&, bool)>("feather_ops::rms_norm_backward");
    return call.call(grad_y, grad_h, h, weight, rstd, need_weight);
}

// A gradient as the kernels read it: each row's values side by side (a broadcast one is copied out).
Tensor as_rows(const Tensor& t) {
    return t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous();
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }

struct SiluMul : public Function<SiluMul> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x) {
        const at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x});
        return silu_mul(x);
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const Tensor x = ctx->get_saved_variables()[0];
        return {silu_mul_backward(as_rows(grads[0]), x)};
    }
};

Tensor silu_mul_autograd(const Tensor& x) {
    if (at::GradMode::is_enabled() && wants_grad(x)) return SiluMul::apply(x);
    const at::AutoDispatchBelowADInplaceOrView below;
    return silu_mul(x);
}

struct RmsNorm : public Function<RmsNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                                 const std::optional<Tensor>& residual, double eps) {
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [y, h, rstd] = rms_norm(x, weight, residual, eps, true);
        const bool add = residual.has_value();
        ctx->set_materialize_grads(false);
        ctx->saved_data["add"] = add;
        ctx->save_for_backward({add ? h : x, weight, rstd});
        ctx->mark_non_differentiable(add ? variable_list{rstd} : variable_list{h, rstd});
        return {y, h, rstd};
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const Tensor& grad_y = grads[0];
        const Tensor& grad_h = grads[1];
        const bool need_x = ctx->needs_input_grad(0);
        const bool need_weight = ctx->needs_input_grad(1);
        const bool need_residual = ctx->saved_data["add"].toBool() && ctx->needs_input_grad(2);
        if (!grad_y.defined())   // only h was used further on
            return {need_x ? grad_h : Tensor(), Tensor(), need_residual ? grad_h : Tensor(), Tensor()};
        const variable_list saved = ctx->get_saved_variables();
        const auto [grad, grad_w] = rms_norm_backward(
            as_rows(grad_y), grad_h.defined() ? std::optional<Tensor>(as_rows(grad_h)) : std::nullopt, as_rows(saved[0]),
            saved[1], saved[2], need_weight);
        return {need_x ? grad : Tensor(), need_weight ? grad_w : Tensor(), need_residual ? grad : Tensor(), Tensor()};
    }
};

Norm rms_norm_autograd(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual, double eps,
                       bool need_rstd) {
    if (at::GradMode::is_enabled() &&
        (wants_grad(x) || wants_grad(weight) || (residual.has_value() && wants_grad(*residual)))) {
        const variable_list out = RmsNorm::apply(x, weight, residual, eps);
        return {out[0], out[1], out[2]};
    }
    const at::AutoDispatchBelowADInplaceOrView below;
    return rms_norm(x, weight, residual, eps, need_rstd);
}

}  // namespace

TORCH_LIBRARY_IMPL(feather_ops, AutogradCUDA, m) {
    m.impl("silu_mul", &silu_mul_autograd);
    m.impl("rms_norm", &rms_norm_autograd);
    // A gradient of a gradient is refused with an error.
    m.impl("silu_mul_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("rms_norm_backward", torch::autograd::autogradNotImplementedFallback());
}
