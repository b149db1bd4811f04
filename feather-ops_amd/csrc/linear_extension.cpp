// The torch ops of the feed-forward operators (include/feather_linear_ops.h). Host code only: each validates its tensors,
// allocates its outputs on their device and calls the C ABI on the current stream. Operands whose rows do not start on 16-byte
// boundaries, or are not whole pieces of 8 values, are refused here and copied by the package.
#include <torch/csrc/stable/library.h>
#include <torch/csrc/stable/ops.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <tuple>

#include "extension_common.h"
#include "feather_internal.h"
#include "feather_linear_ops.h"

namespace {

using torch::stable::Tensor;
using ST = torch::headeronly::ScalarType;

int64_t up_to(int64_t n, int64_t step) { return (n + step - 1) / step * step; }

// A new contiguous [rows, cols]. (Rows that have to be padded are allocated with their padding, the last one's too.)
Tensor new_rows(const Tensor& like, int64_t rows, int64_t cols, int32_t dtype) {
    const int64_t sizes[2] = {rows, cols};
    const int64_t strides[2] = {cols, 1};
    int32_t device_type = 0;
    TORCH_ERROR_CODE_CHECK(aoti_torch_get_device_type(like.get(), &device_type));
    AtenTensorHandle handle = nullptr;
    TORCH_ERROR_CODE_CHECK(
        aoti_torch_empty_strided(2, sizes, strides, dtype, device_type, like.get_device_index(), &handle));
    return Tensor(handle);
}

Tensor new_vector(const Tensor& like, int64_t n, int32_t dtype) {
    const int64_t stride = 1;
    int32_t device_type = 0;
    TORCH_ERROR_CODE_CHECK(aoti_torch_get_device_type(like.get(), &device_type));
    AtenTensorHandle handle = nullptr;
    TORCH_ERROR_CODE_CHECK(
        aoti_torch_empty_strided(1, &n, &stride, dtype, device_type, like.get_device_index(), &handle));
    return Tensor(handle);
}

int half_type(const Tensor& t, const char* name) {
    const auto type = t.scalar_type();
    STD_TORCH_CHECK(type == ST::BFloat16 || type == ST::Half, name, " must be bfloat16 or float16");
    return type == ST::BFloat16 ? FEATHER_BF16 : FEATHER_FP16;
}

int32_t torch_dtype(int type) { return type == FEATHER_BF16 ? aoti_torch_dtype_bfloat16() : aoti_torch_dtype_float16(); }

// A matrix on x's device with its rows' values side by side: its row stride.
int64_t row_stride(const Tensor& t, const char* name) {
    STD_TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
    STD_TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, ".stride(1) must be 1");
    if (t.size(0) <= 1) return t.size(1);
    STD_TORCH_CHECK(t.stride(0) >= t.size(1), name, ".stride(0) must be at least its row length");
    return t.stride(0);
}

// The same of an operand of a product: rows on 16-byte boundaries, whole pieces of 8 values.
int64_t operand_stride(const Tensor& t, const char* name) {
    int64_t ld = row_stride(t, name);
    STD_TORCH_CHECK(t.size(1) % 8 == 0 && ld % 8 == 0 && is_aligned(t.const_data_ptr(), 16), "rows of ", name,
                    " must be whole pieces of 8 values on 16-byte boundaries");
    return ld;
}

void check_device(const Tensor& t, const Tensor& like, const char* name) {
    STD_TORCH_CHECK(t.is_cuda() && t.get_device_index() == like.get_device_index(), name, " must be on x's device");
}

void check_like(const Tensor& t, const Tensor& like, const char* name) {
    check_device(t, like, name);
    STD_TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have x's dtype");
}

const void* check_bias(const std::optional<Tensor>& bias, const Tensor& x, int64_t n) {
    if (!bias.has_value()) return nullptr;
    check_like(*bias, x, "bias");
    STD_TORCH_CHECK(bias->dim() == 1 && bias->size(0) == n && (n <= 1 || bias->stride(0) == 1),
                    "bias must be a contiguous vector of ", n, " values");
    return bias->const_data_ptr();
}

struct Workspace {
    void* data;
    int64_t bytes;
};

Workspace check_workspace(std::optional<Tensor>& workspace, int64_t need, const Tensor& x) {
    STD_TORCH_CHECK(need >= 0, "sizes are out of range");
    if (need == 0) return {nullptr, 0};
    STD_TORCH_CHECK(workspace.has_value() && workspace->is_cuda() && workspace->get_device_index() == x.get_device_index() &&
                        workspace->scalar_type() == ST::Byte && workspace->is_contiguous() && workspace->numel() >= need &&
                        is_aligned(workspace->const_data_ptr(), 256),
                    "a contiguous uint8 workspace of at least ", need, " bytes on x's device is needed, 256-byte aligned");
    return {workspace->mutable_data_ptr(), workspace->numel()};
}

float* floats(Tensor& t) { return static_cast<float*>(t.mutable_data_ptr()); }

// Rows of x as a large product reads them: where neither operand's rows start on half lines of memory, each stage of each row
// costs a line more, and x is copied to whole lines first (4096 x 2576 -> 8192 in 256 x 256 tiles 171 us, with either operand
// copied 138; the copy 9).
constexpr int64_t kHalfLine = 32;   // values

struct Rows {
    Tensor own;
    const void* data;
    int64_t ld;
};

Rows on_lines(const Tensor& x, int64_t ldx, int64_t other_ld, int64_t n, hipStream_t stream) {
    const int64_t m = x.size(0), k = x.size(1);
    if (ldx % kHalfLine == 0 || other_ld % kHalfLine == 0 || m < 512 || n < 2048 || k < 256) return {x, x.const_data_ptr(), ldx};
    const int64_t ld = up_to(k, 2 * kHalfLine);
    Tensor own = new_rows(x, m, ld, torch_dtype(half_type(x, "x")));
    check_launch(feather_copy_rows(x.const_data_ptr(), ldx, own.mutable_data_ptr(), ld, m, k, stream), "copy of rows");
    return {own, own.const_data_ptr(), ld};
}

// feather_ops::gated_forward (feather_gated_linear): (y, what the backward needs), the latter empty unless `keep`.
std::tuple<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                                         const int64_t activation, const bool keep, std::optional<Tensor> workspace) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int type = half_type(x, "x");
    check_like(weight, x, "weight");
    const int64_t ldx = operand_stride(x, "x");
    const int64_t ldw = operand_stride(weight, "weight");
    const int64_t M = x.size(0);
    const int64_t K = x.size(1);
    STD_TORCH_CHECK(weight.size(0) % 2 == 0 && weight.size(1) == K, "weight must be [2 F, ", K, "]: the gates' rows, then the others'");
    const int64_t F = weight.size(0) / 2;
    STD_TORCH_CHECK(M > 0 && F > 0 && K > 0, "x and weight must not be empty");
    STD_TORCH_CHECK(activation >= 0 && activation <= 2, "unknown activation");
    const void* const bias_data = check_bias(bias, x, 2 * F);
    const Workspace ws = check_workspace(workspace, feather_gated_linear_workspace_bytes(M, F, K), x);
    const int64_t ld_kept = 2 * up_to(F, 8);
    Tensor y = new_rows(x, M, F, torch_dtype(type));
    Tensor kept = keep ? new_rows(x, M, ld_kept, aoti_torch_dtype_float32()) : new_rows(x, 0, 0, aoti_torch_dtype_float32());
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    const hipStream_t stream = current_stream(x.get_device_index());
    const Rows rows = on_lines(x, ldx, ldw, 2 * F, stream);
    check_launch(feather_gated_linear(rows.data, rows.ld, weight.const_data_ptr(), ldw, bias_data, type,
                                      static_cast<int>(activation), y.mutable_data_ptr(), F, keep ? floats(kept) : nullptr, ld_kept,
                                      M, F, K, ws.data, ws.bytes, stream),
                 "gated_linear");
    return {y, kept};
}

// feather_ops::gated_backward: the gradients of x, weight and bias, those asked for (the others empty).
std::tuple<Tensor, Tensor, Tensor> gated_backward(const Tensor& grad_y, const Tensor& kept, const Tensor& x, const Tensor& weight,
                                                  const int64_t activation, const bool need_x, const bool need_weight,
                                                  const bool need_bias, std::optional<Tensor> workspace) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int type = half_type(x, "x");
    check_like(weight, x, "weight");
    check_like(grad_y, x, "grad_y");
    const int64_t ldx = operand_stride(x, "x");
    const int64_t ldw = operand_stride(weight, "weight");
    const int64_t M = x.size(0);
    const int64_t K = x.size(1);
    const int64_t F = weight.size(0) / 2;
    STD_TORCH_CHECK(weight.size(0) % 2 == 0 && weight.size(1) == K, "weight must be [2 F, ", K, "]");
    STD_TORCH_CHECK(M > 0 && F > 0 && K > 0, "x and weight must not be empty");
    STD_TORCH_CHECK(grad_y.dim() == 2 && grad_y.size(0) == M && grad_y.size(1) == F, "grad_y must have the output's shape");
    const int64_t ld_kept = 2 * up_to(F, 8);
    check_device(kept, x, "kept");
    STD_TORCH_CHECK(kept.scalar_type() == ST::Float && kept.dim() == 2 && kept.size(0) == M && kept.size(1) == ld_kept &&
                        kept.is_contiguous(),
                    "kept must be what the forward kept");
    STD_TORCH_CHECK(activation >= 0 && activation <= 2, "unknown activation");
    const int32_t dtype = torch_dtype(type);
    const int64_t ld_grad = up_to(2 * F, 2 * kHalfLine);
    Tensor grad = new_rows(x, M, ld_grad, dtype);
    const int64_t parts = feather_gated_backward_parts(M, F);
    Tensor sums = new_rows(x, need_bias ? parts : 0, need_bias ? 2 * F : 0, aoti_torch_dtype_float32());
    Tensor grad_x = new_rows(x, need_x ? M : 0, need_x ? K : 0, dtype);
    Tensor grad_w = new_rows(x, need_weight ? 2 * F : 0, need_weight ? K : 0, dtype);
    Tensor grad_b = new_vector(x, need_bias ? 2 * F : 0, dtype);
    int64_t need = 0;
    if (need_x) need = std::max(need, feather_product_workspace_bytes(M, K, 2 * F));
    if (need_weight) need = std::max(need, feather_product_workspace_bytes(2 * F, K, M));
    const Workspace ws = check_workspace(workspace, need, x);
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    const hipStream_t stream = current_stream(x.get_device_index());
    check_launch(feather_gated_backward(grad_y.const_data_ptr(), row_stride(grad_y, "grad_y"),
                                        static_cast<const float*>(kept.const_data_ptr()), ld_kept, type,
                                        static_cast<int>(activation), grad.mutable_data_ptr(), ld_grad,
                                        need_bias ? floats(sums) : nullptr, M, F, stream),
                 "gated_linear's backward");
    if (need_x)
        check_launch(feather_product(grad.const_data_ptr(), ld_grad, false, weight.const_data_ptr(), ldw, true, nullptr, type,
                                     grad_x.mutable_data_ptr(), K, M, K, 2 * F, ws.data, ws.bytes, stream),
                     "gated_linear's backward");
    if (need_weight)
        check_launch(feather_product(grad.const_data_ptr(), ld_grad, true, x.const_data_ptr(), ldx, true, nullptr, type,
                                     grad_w.mutable_data_ptr(), K, 2 * F, K, M, ws.data, ws.bytes, stream),
                     "gated_linear's backward");
    if (need_bias)
        check_launch(feather_sum_rows(floats(sums), grad_b.mutable_data_ptr(), type, parts, 2 * F, stream),
                     "gated_linear's backward");
    return {grad_x, grad_w, grad_b};
}

// ---- 4-bit weights ----

struct Int4 {
    const uint8_t* codes;
    const void* scale;
    const uint8_t* zero;
    int64_t ld_codes, ld_scale, ld_zero, rows;
    int group;
};

// The group size of K columns in `groups` groups.
int group_of(int64_t K, int64_t groups) {
    for (const int group : {32, 64, 128})
        if (up_to(K, group) / group == groups) return group;
    STD_TORCH_CHECK(false, "scale must have one column for each group of 32, 64 or 128 columns of ", K, ", got ", groups);
    return 0;
}

// Scales [rows, groups] or zero points, stored group by group: the distance of the groups.
int64_t group_stride(const Tensor& t, int64_t rows, const char* name) {
    STD_TORCH_CHECK(rows <= 1 || t.stride(0) == 1, name, " must be stored group by group");
    const int64_t ld = t.size(1) <= 1 ? std::max(rows, t.stride(1)) : t.stride(1);
    STD_TORCH_CHECK(ld >= 4, name, " must have 4 values to a group");
    return ld;
}

Int4 check_int4(const Tensor& codes, const Tensor& scale, const std::optional<Tensor>& zero, int64_t K, const Tensor& like) {
    check_device(codes, like, "codes");
    STD_TORCH_CHECK(codes.scalar_type() == ST::Byte && codes.dim() == 2 && codes.size(1) == (K + 1) / 2,
                    "codes must be uint8 [N, ", (K + 1) / 2, "], two columns to a byte");
    Int4 w{};
    w.rows = codes.size(0);
    w.ld_codes = row_stride(codes, "codes");
    if (w.rows <= 1) w.ld_codes = up_to(w.ld_codes, 4);
    STD_TORCH_CHECK(w.ld_codes % 4 == 0 && is_aligned(codes.const_data_ptr(), 4), "rows of codes must start on 4-byte boundaries");
    check_device(scale, like, "scale");
    STD_TORCH_CHECK(scale.dim() == 2 && scale.size(0) == w.rows, "scale must be [N, groups]");
    w.group = group_of(K, scale.size(1));
    w.ld_scale = group_stride(scale, w.rows, "scale");
    w.codes = static_cast<const uint8_t*>(codes.const_data_ptr());
    w.scale = scale.const_data_ptr();
    if (zero.has_value()) {
        check_device(*zero, like, "zero");
        STD_TORCH_CHECK(zero->scalar_type() == ST::Byte && zero->dim() == 2 && zero->size(0) == w.rows &&
                            zero->size(1) == scale.size(1),
                        "zero must be uint8 with scale's shape");
        w.ld_zero = group_stride(*zero, w.rows, "zero");
        w.zero = static_cast<const uint8_t*>(zero->const_data_ptr());
    }
    return w;
}

// The weight [N, K] in 16 bits, rows a multiple of `pitch` (of 8) values apart.
Tensor new_dequantized(const Int4& w, const Tensor& like, int64_t K, int64_t pitch, int type, hipStream_t stream) {
    const int64_t ld = up_to(K, pitch);
    Tensor out = new_rows(like, w.rows, ld, torch_dtype(type));
    check_launch(feather_int4_dequantize(w.codes, w.ld_codes, w.scale, w.ld_scale, w.zero, w.ld_zero, w.group, type,
                                         out.mutable_data_ptr(), ld, w.rows, K, stream),
                 "dequantize_int4");
    return out;
}

// feather_ops::int4_forward: x [M, K padded with zeros to a multiple of 8] times the weight of K columns.
Tensor int4_forward(const Tensor& x, const Tensor& codes, const Tensor& scale, const std::optional<Tensor>& zero,
                    const std::optional<Tensor>& bias, const int64_t K, const bool gated, const int64_t activation,
                    std::optional<Tensor> workspace) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int type = half_type(x, "x");
    const int64_t ldx = operand_stride(x, "x");
    const int64_t M = x.size(0);
    STD_TORCH_CHECK(K > 0 && x.size(1) == up_to(K, 8), "x must have ", K, " columns, padded to a multiple of 8");
    const Int4 w = check_int4(codes, scale, zero, K, x);
    STD_TORCH_CHECK(scale.scalar_type() == x.scalar_type(), "scale must have x's dtype");
    STD_TORCH_CHECK(M > 0 && w.rows > 0 && (!gated || w.rows % 2 == 0), "x and the weight must not be empty, a gated weight has 2 F rows");
    STD_TORCH_CHECK(activation >= 0 && activation <= 2, "unknown activation");
    const int64_t N = gated ? w.rows / 2 : w.rows;
    const void* const bias_data = check_bias(bias, x, w.rows);
    Tensor y = new_rows(x, M, N, torch_dtype(type));
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    const hipStream_t stream = current_stream(x.get_device_index());
    if (feather_int4_linear_direct(w.codes, w.ld_codes, M, N, K, gated)) {
        const Workspace ws = check_workspace(workspace, feather_int4_linear_workspace_bytes(M, N, K, gated), x);
        check_launch(feather_int4_linear(x.const_data_ptr(), ldx, w.codes, w.ld_codes, w.scale, w.ld_scale, w.zero, w.ld_zero,
                                         w.group, bias_data, type, gated, static_cast<int>(activation), y.mutable_data_ptr(), N, M,
                                         N, K, ws.data, ws.bytes, stream),
                     "int4_linear");
        return y;
    }
    const int64_t K8 = up_to(K, 8);
    const int64_t ldw = up_to(K, 2 * kHalfLine);
    const Tensor full = new_dequantized(w, x, K, 2 * kHalfLine, type, stream);
    if (gated) {
        const Workspace ws = check_workspace(workspace, feather_gated_linear_workspace_bytes(M, N, K8), x);
        check_launch(feather_gated_linear(x.const_data_ptr(), ldx, full.const_data_ptr(), ldw, bias_data, type,
                                          static_cast<int>(activation), y.mutable_data_ptr(), N, nullptr, 0, M, N, K8, ws.data,
                                          ws.bytes, stream),
                     "int4_linear");
    } else {
        const Workspace ws = check_workspace(workspace, feather_product_workspace_bytes(M, N, K8), x);
        check_launch(feather_product(x.const_data_ptr(), ldx, false, full.const_data_ptr(), ldw, false, bias_data, type,
                                     y.mutable_data_ptr(), N, M, N, K8, ws.data, ws.bytes, stream),
                     "int4_linear");
    }
    return y;
}

// feather_ops::int4_backward: dx = dy W, [M, K], with W rounded to dy's type. dy's rows are padded with zeros.
Tensor int4_backward(const Tensor& grad_y, const Tensor& codes, const Tensor& scale, const std::optional<Tensor>& zero,
                     const int64_t K, std::optional<Tensor> workspace) {
    STD_TORCH_CHECK(grad_y.is_cuda(), "grad_y must be a CUDA tensor");
    const int type = half_type(grad_y, "grad_y");
    const int64_t ld = operand_stride(grad_y, "grad_y");
    const int64_t M = grad_y.size(0);
    const Int4 w = check_int4(codes, scale, zero, K, grad_y);
    STD_TORCH_CHECK(scale.scalar_type() == grad_y.scalar_type(), "scale must have grad_y's dtype");
    STD_TORCH_CHECK(M > 0 && K > 0 && w.rows > 0 && grad_y.size(1) == up_to(w.rows, 8), "grad_y must have the output's shape");
    const Workspace ws = check_workspace(workspace, feather_product_workspace_bytes(M, K, w.rows), grad_y);
    Tensor grad_x = new_rows(grad_y, M, K, torch_dtype(type));
    torch::stable::accelerator::DeviceGuard guard(grad_y.get_device_index());
    const hipStream_t stream = current_stream(grad_y.get_device_index());
    const Tensor full = new_dequantized(w, grad_y, K, 2 * kHalfLine, type, stream);
    check_launch(feather_product(grad_y.const_data_ptr(), ld, false, full.const_data_ptr(), up_to(K, 2 * kHalfLine), true, nullptr, type,
                                 grad_x.mutable_data_ptr(), K, M, K, w.rows, ws.data, ws.bytes, stream),
                 "int4_linear's backward");
    return grad_x;
}

// feather_ops::int4_quantize (feather_int4_quantize): (codes [N, bytes to a multiple of 16], scale [groups, N to a multiple of 4],
// zero, the same or empty).
std::tuple<Tensor, Tensor, Tensor> int4_quantize(const Tensor& w, const int64_t group, const bool zeros) {
    STD_TORCH_CHECK(w.is_cuda(), "weight must be a CUDA tensor");
    const int type = half_type(w, "weight");
    const int64_t ldw = row_stride(w, "weight");
    const int64_t N = w.size(0);
    const int64_t K = w.size(1);
    STD_TORCH_CHECK(group == 32 || group == 64 || group == 128, "a group has 32, 64 or 128 columns, got ", group);
    STD_TORCH_CHECK(N > 0 && K > 0, "weight must not be empty");
    const int64_t groups = up_to(K, group) / group;
    const int64_t ld = up_to(N, 4);
    const int64_t bytes = up_to((K + 1) / 2, 16);   // rows on 16-byte boundaries
    Tensor codes = new_rows(w, N, bytes, aoti_torch_dtype_uint8());
    Tensor scale = new_rows(w, groups, ld, torch_dtype(type));
    Tensor zero = new_rows(w, zeros ? groups : 0, zeros ? ld : 0, aoti_torch_dtype_uint8());
    torch::stable::accelerator::DeviceGuard guard(w.get_device_index());
    check_launch(feather_int4_quantize(w.const_data_ptr(), ldw, type, static_cast<int>(group),
                                       static_cast<uint8_t*>(codes.mutable_data_ptr()), bytes, scale.mutable_data_ptr(), ld,
                                       zeros ? static_cast<uint8_t*>(zero.mutable_data_ptr()) : nullptr, ld, N, K,
                                       current_stream(w.get_device_index())),
                 "quantize_int4");
    return {codes, scale, zero};
}

// feather_ops::int4_dequantize (feather_int4_dequantize): [N, K to a multiple of 8] in scale's dtype.
Tensor int4_dequantize(const Tensor& codes, const Tensor& scale, const std::optional<Tensor>& zero, const int64_t K) {
    STD_TORCH_CHECK(codes.is_cuda(), "codes must be a CUDA tensor");
    const int type = half_type(scale, "scale");
    const Int4 w = check_int4(codes, scale, zero, K, codes);
    STD_TORCH_CHECK(w.rows > 0 && K > 0, "the weight must not be empty");
    torch::stable::accelerator::DeviceGuard guard(codes.get_device_index());
    return new_dequantized(w, codes, K, 8, type, current_stream(codes.get_device_index()));
}

}  // namespace

STABLE_TORCH_LIBRARY_FRAGMENT(feather_ops, m) {
    m.def(
        "gated_forward(Tensor x, Tensor weight, Tensor? bias, int activation, bool keep, Tensor(a!)? workspace) -> (Tensor, "
        "Tensor)");
    m.def(
        "gated_backward(Tensor grad_y, Tensor kept, Tensor x, Tensor weight, int activation, bool need_x, bool need_weight, "
        "bool need_bias, Tensor(a!)? workspace) -> (Tensor, Tensor, Tensor)");
    m.def(
        "int4_forward(Tensor x, Tensor codes, Tensor scale, Tensor? zero, Tensor? bias, int k, bool gated, int activation, "
        "Tensor(a!)? workspace) -> Tensor");
    m.def("int4_backward(Tensor grad_y, Tensor codes, Tensor scale, Tensor? zero, int k, Tensor(a!)? workspace) -> Tensor");
    m.def("int4_quantize(Tensor weight, int group, bool zeros) -> (Tensor, Tensor, Tensor)");
    m.def("int4_dequantize(Tensor codes, Tensor scale, Tensor? zero, int k) -> Tensor");
}

STABLE_TORCH_LIBRARY_IMPL(feather_ops, CUDA, m) {
    m.impl("gated_forward", TORCH_BOX(&gated_forward));
    m.impl("gated_backward", TORCH_BOX(&gated_backward));
    m.impl("int4_forward", TORCH_BOX(&int4_forward));
    m.impl("int4_backward", TORCH_BOX(&int4_backward));
    m.impl("int4_quantize", TORCH_BOX(&int4_quantize));
    m.impl("int4_dequantize", TORCH_BOX(&int4_dequantize));
}
