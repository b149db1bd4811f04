// The gated block and the 4-bit product as nodes of torch's autograd graph, in C++ for the reason that block_autograd.cpp gives.
#include "autograd_common.h"

#include <cstdint>
#include <optional>
#include <tuple>

namespace {

using namespace feather;

std::tuple<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                                         int64_t activation, bool keep, const std::optional<Tensor>& workspace) {
    static const auto call =
        op<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const std::optional<Tensor>&, int64_t, bool,
                                      const std::optional<Tensor>&)>("feather_ops::gated_forward");
    return call.call(x, weight, bias, activation, keep, workspace);
}

std::tuple<Tensor, Tensor, Tensor> gated_backward(const Tensor& grad_y, const Tensor& kept, const Tensor& x, const Tensor& weight,
                                                  int64_t activation, bool need_x, bool need_weight, bool need_bias,
                                                  const std::optional<Tensor>& workspace) {
    static const auto call =
        op<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t, bool, bool,
                                              bool, const std::optional<Tensor>&)>("feather_ops::gated_backward");
    return call.call(grad_y, kept, x, weight, activation, need_x, need_weight, need_bias, workspace);
}

Tensor int4_forward(const Tensor& x, const Tensor& codes, const Tensor& scale, const std::optional<Tensor>& zero,
                    const std::optional<Tensor>& bias, int64_t k, bool gated, int64_t activation,
                    const std::optional<Tensor>& workspace) {
    static const auto call =
        op<Tensor(const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&, const std::optional<Tensor>&, int64_t,
                  bool, int64_t, const std::optional<Tensor>&)>("feather_ops::int4_forward");
    return call.call(x, codes, scale, zero, bias, k, gated, activation, workspace);
}

Tensor int4_backward(const Tensor& grad_y, const Tensor& codes, const Tensor& scale, const std::optional<Tensor>& zero, int64_t k,
                     const std::optional<Tensor>& workspace) {
    static const auto call = op<Tensor(const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&, int64_t,
                                       const std::optional<Tensor>&)>("feather_ops::int4_backward");
    return call.call(grad_y, codes, scale, zero, k, workspace);
}

// The column sums of each 128 rows, and their sum: of the reductions here, ones that a captured graph can hold.
Tensor column_sums(const Tensor& t) {
    using Tiles = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
    static const auto tiles = op<Tiles(const Tensor&, bool, bool, bool, bool, bool)>("feather_ops::quantize_tiles");
    static const auto sum = op<Tensor(const Tensor&, int64_t)>("feather_ops::sum_rows");
    return sum.call(std::get<4>(tiles.call(t, false, false, false, false, true)), t.scalar_type() == at::kBFloat16 ? 0 : 1);
}

// A gradient as an operand of a product: rows on 16-byte boundaries, of whole pieces of 8 values, zeros behind the last.
Tensor as_operand(const Tensor& t) {
    const int64_t cols = t.size(1);
    const bool fake = t.key_set().has(c10::DispatchKey::Python);
    if (cols % 8 == 0 && t.stride(1) == 1 && t.stride(0) >= cols && t.stride(0) % 8 == 0 && t.stride(0) <= int64_t{1} << 21 &&
        (fake || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0))
        return t;
    const int64_t whole = (cols + 7) / 8 * 8;
    Tensor out = at::empty({t.size(0), whole}, t.options());
    out.narrow(1, 0, cols).copy_(t);
    if (whole > cols) out.narrow(1, cols, whole - cols).zero_();
    return out;
}

// y = act(x Wg^T + bg) * (x Wu^T + bu). Both sums are kept in fp32: rounded to bf16 they make the gradients' error, 2.34e-3 of
// their norm, 2.96e-3 (512 x 512 -> 512, computed in 64 bits). They cost 80 us forward and as much backward of the 1920 of 4096 x
// 4096 -> 12288.
struct GatedLinear : public Function<GatedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                          int64_t activation, const std::optional<Tensor>& workspace) {
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [y, kept] = gated_forward(x, weight, bias, activation, true, workspace);
        ctx->save_for_backward({kept, x, weight});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["bias"] = bias.has_value();
        if (workspace.has_value()) ctx->saved_data["workspace"] = *workspace;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const bool need_x = ctx->needs_input_grad(0);
        const bool need_w = ctx->needs_input_grad(1);
        const bool bias = ctx->saved_data["bias"].toBool();
        const bool need_b = bias && ctx->needs_input_grad(2);
        const variable_list saved = ctx->get_saved_variables();
        refuse_tangents("gated_linear", {grads[0]});
        refuse_foreign_streams("gated_linear", grads[0]);
        const bool twice = at::GradMode::is_enabled();
        const at::NoGradGuard once;
        auto [grad_x, grad_w, grad_b] =
            gated_backward(as_rows(grads[0]), saved[0], saved[1], saved[2], ctx->saved_data["activation"].toInt(), need_x, need_w,
                           need_b, workspace_of(ctx->saved_data["workspace"]));
        if (!need_x) grad_x = Tensor();
        if (!need_w) grad_w = Tensor();
        if (!need_b) grad_b = Tensor();
        if (twice) {   // each depends on x, the weight and the bias, by the slope, and on dy
            const auto node = torch::autograd::get_current_node();
            TORCH_CHECK(node, "gated_linear: its backward runs outside of its node");
            const torch::autograd::Edge last = bias ? node->next_edge(2) : torch::autograd::Edge();
            for (Tensor* grad : {&grad_x, &grad_w, &grad_b})
                refuse_second("gated_linear", *grad, grads[0], {node->next_edge(0), node->next_edge(1), last});
        }
        return {grad_x, grad_w, grad_b, Tensor(), Tensor()};
    }
};

// feather_ops::gated_linear, for matrices with rows on 16-byte boundaries, of whole pieces of 8 values; workspace: enough for every
// product that is taken.
Tensor gated_linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, int64_t activation,
                    const std::optional<Tensor>& workspace) {
    refuse_tangents("gated_linear", {x, weight, bias});
    if (at::GradMode::is_enabled() &&
        (wants_grad(x) || wants_grad(weight) || (bias.has_value() && wants_grad(*bias))))
        return GatedLinear::apply(x, weight, bias, activation, workspace);
    return std::get<0>(gated_forward(x, weight, bias, activation, false, workspace));
}

// y = x W^T + bias with a frozen 4-bit weight: dx = dy W.
struct Int4Linear : public Function<Int4Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scale,
                          const std::optional<Tensor>& zero, const std::optional<Tensor>& bias, int64_t k,
                          const std::optional<Tensor>& workspace) {
        const at::AutoDispatchBelowADInplaceOrView below;
        Tensor y = int4_forward(x, codes, scale, zero, bias, k, false, 0, workspace);
        ctx->save_for_backward({codes, scale, zero.has_value() ? *zero : Tensor()});
        ctx->saved_data["k"] = k;
        ctx->saved_data["x_cols"] = x.size(1);
        ctx->saved_data["bias"] = bias.has_value();
        if (workspace.has_value()) ctx->saved_data["workspace"] = *workspace;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        const bool need_x = ctx->needs_input_grad(0);
        // operands that are not there are not counted
        const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(saved[2].defined() ? 4 : 3);
        refuse_tangents("int4_linear", {grads[0]});
        refuse_foreign_streams("int4_linear", grads[0]);
        const bool twice = at::GradMode::is_enabled();
        const at::NoGradGuard once;
        Tensor grad_x, grad_b;
        if (need_x) {
            const int64_t k = ctx->saved_data["k"].toInt();
            const int64_t cols = ctx->saved_data["x_cols"].toInt();
            grad_x = int4_backward(as_operand(grads[0]), saved[0], saved[1],
                                   saved[2].defined() ? std::optional<Tensor>(saved[2]) : std::nullopt, k,
                                   workspace_of(ctx->saved_data["workspace"]));
            if (cols > k) grad_x = at::constant_pad_nd(grad_x, {0, cols - k});   // x's padding
        }
        if (need_b) grad_b = column_sums(as_rows(grads[0]));
        if (twice) {
            refuse_second("int4_linear", grad_x, grads[0], {});
            refuse_second("int4_linear", grad_b, grads[0], {});
        }
        return {grad_x, Tensor(), Tensor(), Tensor(), grad_b, Tensor(), Tensor()};
    }
};

// feather_ops::int4_linear, for x as int4_forward takes it.
Tensor int4_linear(const Tensor& x, const Tensor& codes, const Tensor& scale, const std::optional<Tensor>& zero,
                   const std::optional<Tensor>& bias, int64_t k, const std::optional<Tensor>& workspace) {
    refuse_tangents("int4_linear", {x, scale, bias});
    if (at::GradMode::is_enabled() && (wants_grad(x) || (bias.has_value() && wants_grad(*bias))))
        return Int4Linear::apply(x, codes, scale, zero, bias, k, workspace);
    return int4_forward(x, codes, scale, zero, bias, k, false, 0, workspace);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(feather_ops, m) {
    m.def(
        "gated_linear(Tensor x, Tensor weight, Tensor? bias, int activation, Tensor(a!)? workspace) -> Tensor",
        &gated_linear);
    m.def(
        "int4_linear(Tensor x, Tensor codes, Tensor scale, Tensor? zero, Tensor? bias, int k, Tensor(a!)? workspace) -> Tensor",
        &int4_linear);
}
