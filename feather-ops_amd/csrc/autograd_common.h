// What the autograd nodes share (block_autograd.cpp, linear_autograd.cpp).
#pragma once

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/inductor/aoti_torch/c/shim.h>
#include <torch/library.h>

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <memory>
#include <optional>
#include <string>
#include <tuple>
#include <utility>

namespace feather {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

template <typename Signature>
c10::TypedOperatorHandle<Signature> op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

// A gradient as the kernels read it: each row's values side by side (a broadcast one is copied out).
inline Tensor as_rows(const Tensor& t) {
    return t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous();
}

inline bool wants_grad(const Tensor& t) { return t.requires_grad(); }

// Forward mode has no formulas here: an operand's tangent is refused, with and without a graph, and never dropped. (Under a
// transform the op is called once more for each level, with that level's tangents.)
inline void refuse_tangents(const char* name, std::initializer_list<std::optional<Tensor>> operands) {
    for (const auto& t : operands)
        TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t), "forward-mode derivatives of ", name,
                                    " are not implemented");
}

// The forward's workspace for the backward's products: both run on the forward's stream. A graph that captures the backward
// gets one of its own, whose arrival counters each replay clears, as graphs may share the memory of what a capture frees.
inline std::optional<Tensor> workspace_of(const c10::IValue& kept) {
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

// Whether a stream is being captured. (The default one cannot be.)
inline bool is_capturing(const c10::Stream& stream) {
    if (stream.id() == 0) return false;
    const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
    const c10::Stream before = guard.exchangeStream(stream);
    void* handle = nullptr;
    const bool known = aoti_torch_get_current_cuda_stream(stream.device_index(), &handle) == AOTI_TORCH_SUCCESS;
    guard.exchangeStream(before);
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    return known && hipStreamIsCapturing(static_cast<hipStream_t>(handle), &capture) == hipSuccess &&
           capture == hipStreamCaptureStatusActive;
}

// What runs after `node` in this backward, up to `depth` nodes on, on a stream that is neither `current` nor captured itself.
inline bool leads_astray(const torch::autograd::Node& node, const c10::Stream& current, int depth) {
    const auto* const runs = torch::autograd::get_current_graph_task_exec_info();
    for (const torch::autograd::Edge& edge : node.next_edges()) {
        if (!edge.is_valid()) continue;
        if (runs && !runs->empty()) {
            const auto found = runs->find(edge.function.get());
            if (found == runs->end() || !found->second.should_execute()) continue;
        }
        const std::optional<c10::Stream> stream = edge.function->stream();
        if (stream && *stream != current && !is_capturing(*stream)) return true;
        if (depth > 1 && leads_astray(*edge.function, current, depth - 1)) return true;
    }
    return false;
}

// A backward that is being captured hands its gradients to the nodes before it on their streams. A leaf's node lives as long as
// any graph on it, on the stream where that graph began: where that is not being captured, the wait between the two would end
// the capture, and with it the process. It is refused instead. (Between the operator and a leaf there are the package's own views,
// casts and copies: three at most.)
inline void refuse_foreign_streams(const char* name, const Tensor& grad_y) {
    const auto node = torch::autograd::get_current_node();
    if (!node || !grad_y.is_cuda() || grad_y.key_set().has(c10::DispatchKey::Python)) return;
    const c10::Stream current = c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getStream(grad_y.device());
    TORCH_CHECK(!is_capturing(current) || !leads_astray(*node, current, 4), name,
                ": its backward is being captured, and an operand belongs to a graph that lives on another stream, such as an "
                "earlier pass's loss. Release that graph, or run that pass on the capturing stream");
}

// Makes `grad` depend on what it was computed from, by way of a node that refuses to go on: the gradient that came in and
// operands, by the edges that the forward's node has to them (they need not be kept themselves).
inline void refuse_second(const char* name, Tensor& grad, const Tensor& grad_y,
                          std::initializer_list<torch::autograd::Edge> operands) {
    torch::autograd::edge_list from;
    if (grad_y.requires_grad()) from.push_back(torch::autograd::impl::gradient_edge(grad_y));
    for (const auto& operand : operands)
        if (operand.is_valid()) from.push_back(operand);
    if (!grad.defined() || from.empty()) return;
    torch::autograd::set_history(grad, std::make_shared<torch::autograd::Error>(
                                           std::string("second derivatives of ") + name + " are not implemented",
                                           std::move(from)));
}

}  // namespace feather
