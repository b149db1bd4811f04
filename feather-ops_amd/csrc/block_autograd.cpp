// The fp8 layer, and the gradients of rms_norm and silu_mul, as nodes of torch's autograd graph, in C++. The backward of a
// CUDA tensor runs on a thread of its own, where a function in Python needs the interpreter's lock. Forward and backward of
// small tensors, whatever their kernels take, in microseconds with such functions / with these nodes: the norm 112 / 87, the
// gate 65-72 / 50, the layer 160 / 132; with one thread for all 51 / 45, 29 / 23 and 88 / 74. A product with a number, a node
// of torch's own, takes 48-51 and 22.
//
// Host code; unlike the ops themselves (block_extension.cpp) it needs torch's C++ interface and not only its stable one, and
// is a library of its own for that.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/inductor/aoti_torch/c/shim.h>
#include <torch/library.h>

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <memory>
#include <optional>
#include <tuple>
#include <utility>

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

using Tiles = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

Tiles quantize_tiles(const Tensor& x, bool e5m2, bool square, bool plain, bool transposed, bool sums) {
    static const auto call = op<Tiles(const Tensor&, bool, bool, bool, bool, bool)>("feather_ops::quantize_tiles");
    return call.call(x, e5m2, square, plain, transposed, sums);
}

std::tuple<Tensor, Tensor> quantize_blocks(const Tensor& x, bool e5m2) {
    static const auto call = op<std::tuple<Tensor, Tensor>(const Tensor&, bool)>("feather_ops::quantize_blocks");
    return call.call(x, e5m2);
}

Tensor sum_rows(const Tensor& part, int64_t out_type) {
    static const auto call = op<Tensor(const Tensor&, int64_t)>("feather_ops::sum_rows");
    return call.call(part, out_type);
}

Tensor block_scaled_mm(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale,
                       const std::optional<Tensor>& bias, int64_t out_type, const std::optional<Tensor>& workspace) {
    static const auto call = op<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&,
                                       int64_t, const std::optional<Tensor>&)>("feather_ops::block_scaled_mm");
    return call.call(a, a_scale, b, b_scale, bias, out_type, workspace);
}

// The C ABI's number of a value type.
int64_t type_number(at::ScalarType type) {
    TORCH_CHECK_VALUE(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat,
                      "values must be bfloat16, float16 or float32");
    return type == at::kBFloat16 ? 0 : type == at::kHalf ? 1 : 2;
}

// A gradient as the kernels read it: each row's values side by side (a broadcast one is copied out).
Tensor as_rows(const Tensor& t) {
    return t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous();
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }

// Forward mode has no formulas here: an operand's tangent is refused, with and without a graph, and never dropped. (Under a
// transform the op is called once more for each level, with that level's tangents.)
void refuse_tangents(const char* name, std::initializer_list<std::optional<Tensor>> operands) {
    for (const auto& t : operands)
        TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t), "forward-mode derivatives of ", name,
                                    " are not implemented");
}

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
    refuse_tangents("silu_mul", {x});
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
    refuse_tangents("rms_norm", {x, weight, residual});
    if (at::GradMode::is_enabled() &&
        (wants_grad(x) || wants_grad(weight) || (residual.has_value() && wants_grad(*residual)))) {
        const variable_list out = RmsNorm::apply(x, weight, residual, eps);
        return {out[0], out[1], out[2]};
    }
    const at::AutoDispatchBelowADInplaceOrView below;
    return rms_norm(x, weight, residual, eps, need_rstd);
}

// The forward's workspace for the backward's products: both run on the forward's stream. A graph that captures the backward
// gets one of its own, whose arrival counters each replay clears, as graphs may share the memory of what a capture frees.
std::optional<Tensor> workspace_of(const c10::IValue& kept) {
    if (!kept.isTensor()) return std::nullopt;
    const Tensor& workspace = kept.toTensor();
    if (workspace.key_set().has(c10::DispatchKey::Python)) return workspace;   // fake
    void* stream = nullptr;
    TORCH_CHECK(aoti_torch_get_current_cuda_stream(workspace.get_device(), &stream) == AOTI_TORCH_SUCCESS,
                "no current stream");
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    TORCH_CHECK(hipStreamIsCapturing(static_cast<hipStream_t>(stream), &capture) == hipSuccess,
                "the stream's capture status is unknown");
    if (capture == hipStreamCaptureStatusNone) return workspace;
    constexpr int64_t kCounterBytes = 64 * 1024;
    Tensor own = at::empty_like(workspace);
    own.narrow(0, 0, std::min(kCounterBytes, own.numel())).zero_();
    return own;
}

// Makes `grad` depend on what it was computed from, by way of a node that refuses to go on: the gradient that came in and an
// operand, by the edge that the layer's node has to it (the operand itself is not kept, its fp8 copies are).
void refuse_second(Tensor& grad, const Tensor& grad_y, const torch::autograd::Edge& operand) {
    torch::autograd::edge_list from;
    if (grad_y.requires_grad()) from.push_back(torch::autograd::impl::gradient_edge(grad_y));
    if (operand.is_valid()) from.push_back(operand);
    if (!grad.defined() || from.empty()) return;
    torch::autograd::set_history(grad, std::make_shared<torch::autograd::Error>(
                                           "second derivatives of block_scaled_linear are not implemented", std::move(from)));
}

// y = x w^T + bias in fp8: x and w quantized by rows and by squares; dx = dy w and dw = dy^T x with dy, dy^T and x^T quantized
// by rows, and w^T by the same squares. What is kept for the backward is fp8.
struct Linear : public Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                          bool e5m2, const std::optional<Tensor>& codes, const std::optional<Tensor>& scale,
                          const std::optional<Tensor>& workspace) {
        const at::AutoDispatchBelowADInplaceOrView below;
        const bool need_x = x.requires_grad();
        const bool need_w = weight.requires_grad();
        const auto [xq, xs, xt, xts, no_sums] = quantize_tiles(x, e5m2, false, true, need_w, false);
        Tensor wq, ws, wt, wts;
        if (codes.has_value()) {
            wq = *codes;
            ws = *scale;
        } else {
            Tensor none;
            std::tie(wq, ws, wt, wts, none) = quantize_tiles(weight, e5m2, true, true, need_x, false);
        }
        Tensor y = block_scaled_mm(xq, xs, wq, ws, bias, type_number(x.scalar_type()), workspace);
        // A weight quantized before the call is not kept transposed: the backward quantizes it again.
        const bool again = need_x && codes.has_value();
        ctx->save_for_backward({need_w ? xt : Tensor(), need_w ? xts : Tensor(), need_x && !again ? wt : Tensor(),
                                need_x && !again ? wts : Tensor(), again ? weight : Tensor()});
        ctx->saved_data["e5m2"] = e5m2;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["x_type"] = type_number(x.scalar_type());
        ctx->saved_data["w_type"] = type_number(weight.scalar_type());
        if (workspace.has_value()) ctx->saved_data["workspace"] = *workspace;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const bool need_x = ctx->needs_input_grad(0);
        const bool need_w = ctx->needs_input_grad(1);
        const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
        const bool e5m2 = ctx->saved_data["e5m2"].toBool();
        const int64_t x_type = ctx->saved_data["x_type"].toInt();
        const variable_list saved = ctx->get_saved_variables();
        refuse_tangents("block_scaled_linear", {grads[0]});
        const bool twice = at::GradMode::is_enabled();
        const at::NoGradGuard once;
        const std::optional<Tensor> workspace = workspace_of(ctx->saved_data["workspace"]);
        const auto [gq, gs, gt, gts, sums] = quantize_tiles(as_rows(grads[0]), e5m2, false, need_x, need_w, need_b);
        Tensor grad_x, grad_w, grad_b;
        if (need_x) {
            Tensor wt = saved[2];
            Tensor wts = saved[3];
            if (saved[4].defined()) {
                Tensor none, none_scale, no_sums;
                std::tie(none, none_scale, wt, wts, no_sums) =
                    quantize_tiles(saved[4].detach(), e5m2, true, false, true, false);
            }
            grad_x = block_scaled_mm(gq, gs, wt, wts, std::nullopt, x_type, workspace);
        }
        if (need_w)
            grad_w = block_scaled_mm(gt, gts, saved[0], saved[1], std::nullopt, ctx->saved_data["w_type"].toInt(), workspace);
        if (need_b) grad_b = sum_rows(sums, x_type);
        if (twice) {   // dx depends on the weight, dW on x, all three on dy
            const auto node = torch::autograd::get_current_node();
            TORCH_CHECK(node, "block_scaled_linear: its backward runs outside of its node");
            refuse_second(grad_x, grads[0], node->next_edge(1));
            refuse_second(grad_w, grads[0], node->next_edge(0));
            refuse_second(grad_b, grads[0], {});
        }
        return {grad_x, grad_w, grad_b, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// feather_ops::block_scaled_linear, for matrices x and weight: weight_codes and weight_scale, the weight's squares, where
// they are there already; bias in x's dtype; workspace as block_scaled_mm's, enough for every product that is taken.
Tensor block_scaled_linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, bool e5m2,
                           const std::optional<Tensor>& weight_codes, const std::optional<Tensor>& weight_scale,
                           const std::optional<Tensor>& workspace) {
    TORCH_CHECK(weight_codes.has_value() == weight_scale.has_value(), "codes and scale of the weight go together");
    refuse_tangents("block_scaled_linear", {x, weight, bias});
    if (at::GradMode::is_enabled() &&
        (wants_grad(x) || wants_grad(weight) || (bias.has_value() && wants_grad(*bias))))
        return Linear::apply(x, weight, bias, e5m2, weight_codes, weight_scale, workspace);
    const auto [xq, xs] = quantize_blocks(x, e5m2);
    if (weight_codes.has_value())
        return block_scaled_mm(xq, xs, *weight_codes, *weight_scale, bias, type_number(x.scalar_type()), workspace);
    const Tiles w = quantize_tiles(weight, e5m2, true, true, false, false);
    return block_scaled_mm(xq, xs, std::get<0>(w), std::get<1>(w), bias, type_number(x.scalar_type()), workspace);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(feather_ops, m) {
    m.def(
        "block_scaled_linear(Tensor x, Tensor weight, Tensor? bias, bool e5m2, Tensor? weight_codes, Tensor? weight_scale, "
        "Tensor(a!)? workspace) -> Tensor",
        &block_scaled_linear);
}

TORCH_LIBRARY_IMPL(feather_ops, AutogradCUDA, m) {
    m.impl("silu_mul", &silu_mul_autograd);
    m.impl("rms_norm", &rms_norm_autograd);
    // A gradient of a gradient is refused with an error.
    m.impl("silu_mul_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("rms_norm_backward", torch::autograd::autogradNotImplementedFallback());
}
