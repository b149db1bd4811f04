// The torch ops of the operators with one scale for each block of 128 values (include/feather_block_ops.h). Host code
// only: each validates its tensors, allocates its outputs on their device and calls the C ABI on the current stream. The
// codes' rows are padded to multiples of 64 bytes: the product needs 16, and a block that starts inside a half line costs it a
// line more (4096 x 5000 x 2576: rows of 2576 bytes 76 us, 2624 68, 2688 67; 16 x 5000 x 2576: 7.1, 6.7, 8.3). Scales are
// stored block by block ([blocks, rows], handed out as its transpose). Outputs that a call does not ask for come back empty.
#include <torch/csrc/stable/library.h>
#include <torch/csrc/stable/ops.h>

#include <cstdint>
#include <optional>
#include <tuple>

#include "extension_common.h"
#include "feather_block_ops.h"

namespace {

using torch::stable::Tensor;
using ST = torch::headeronly::ScalarType;

constexpr int64_t kBlock = 128;

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

Tensor new_strided(const Tensor& like, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, int32_t dtype) {
    const int64_t sizes[2] = {rows, cols};
    const int64_t strides[2] = {row_stride, col_stride};
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

Tensor new_matrix(const Tensor& like, int64_t rows, int64_t cols, int32_t dtype) {
    return new_strided(like, rows, cols, cols, 1, dtype);
}

int32_t torch_dtype(int type) {
    return type == FEATHER_BF16   ? aoti_torch_dtype_bfloat16()
           : type == FEATHER_FP16 ? aoti_torch_dtype_float16()
                                  : aoti_torch_dtype_float32();
}

int32_t fp8_dtype(bool e5m2) { return e5m2 ? aoti_torch_dtype_float8_e5m2() : aoti_torch_dtype_float8_e4m3fn(); }

int value_type(const Tensor& t, const char* name) {
    const auto type = t.scalar_type();
    STD_TORCH_CHECK(type == ST::BFloat16 || type == ST::Half || type == ST::Float, name,
                    " must be bfloat16, float16 or float32");
    return type == ST::BFloat16 ? FEATHER_BF16 : type == ST::Half ? FEATHER_FP16 : FEATHER_FP32;
}

bool is_e5m2(const Tensor& t, const char* name) {
    const auto type = t.scalar_type();
    STD_TORCH_CHECK(type == ST::Float8_e4m3fn || type == ST::Float8_e5m2, name,
                    " must be float8_e4m3fn or float8_e5m2");
    return type == ST::Float8_e5m2;
}

// A matrix with its rows' values side by side; rows may be apart.
int64_t row_stride(const Tensor& t, const char* name) {
    STD_TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
    STD_TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, ".stride(1) must be 1");
    if (t.size(0) <= 1) return t.size(1);
    STD_TORCH_CHECK(t.stride(0) >= t.size(1), name, ".stride(0) must be at least its row length");
    return t.stride(0);
}

void check_same(const Tensor& t, const Tensor& like, const char* name) {
    STD_TORCH_CHECK(t.is_cuda() && t.get_device_index() == like.get_device_index(), name, " must be on x's device");
    STD_TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have x's dtype");
    STD_TORCH_CHECK(t.dim() == 2 && t.size(0) == like.size(0) && t.size(1) == like.size(1), name,
                    " must have x's shape");
}

void check_weight(const Tensor& w, const Tensor& x) {
    STD_TORCH_CHECK(w.is_cuda() && w.get_device_index() == x.get_device_index(), "weight must be on x's device");
    STD_TORCH_CHECK(w.scalar_type() == x.scalar_type() || w.scalar_type() == ST::Float,
                    "weight must have x's dtype or float32");
    STD_TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(1) && (w.size(0) <= 1 || w.stride(0) == 1),
                    "weight must be a contiguous vector of x's row length");
}

struct Codes {
    Tensor codes, scale;
    int64_t ld;
};

// New codes [rows, cols] and scales [scale_rows, ceil(cols / 128)].
Codes new_codes(const Tensor& like, int64_t rows, int64_t cols, int64_t scale_rows, bool e5m2) {
    const int64_t ld = (cols + 63) / 64 * 64;
    return {new_strided(like, rows, cols, ld, 1, fp8_dtype(e5m2)),
            new_strided(like, scale_rows, blocks_of(cols), 1, scale_rows, aoti_torch_dtype_float32()), ld};
}

const float* floats(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }
float* floats(Tensor& t) { return static_cast<float*>(t.mutable_data_ptr()); }
uint8_t* bytes(Tensor& t) { return static_cast<uint8_t*>(t.mutable_data_ptr()); }

// Scales whose rows are at most 2^20 apart, as the product takes them: copied where they are not.
Tensor near_rows(const Tensor& scale) {
    return scale.size(0) > 1 && scale.stride(0) > (1 << 20) ? torch::stable::contiguous(scale) : scale;
}

// feather_ops::block_scaled_mm (feather_block_scaled_mm); out_type: 0 bfloat16, 1 float16, 2 float32. workspace: uint8,
// as scaled_mm_splitk's, where the shape needs one.
Tensor block_scaled_mm(const Tensor& a, Tensor a_scale, const Tensor& b, Tensor b_scale,
                       const std::optional<Tensor>& bias, const int64_t out_type, std::optional<Tensor> workspace) {
    STD_TORCH_CHECK(a.is_cuda() && b.is_cuda() && a_scale.is_cuda() && b_scale.is_cuda(),
                    "a, b and their scales must be CUDA tensors");
    const auto device_index = a.get_device_index();
    STD_TORCH_CHECK(b.get_device_index() == device_index && a_scale.get_device_index() == device_index &&
                        b_scale.get_device_index() == device_index,
                    "a, b and their scales must be on one device");
    const bool a_e5m2 = is_e5m2(a, "a");
    const bool b_e5m2 = is_e5m2(b, "b");
    int64_t lda = row_stride(a, "a");
    int64_t ldb = row_stride(b, "b");
    const int64_t M = a.size(0);
    const int64_t N = b.size(0);
    const int64_t K = a.size(1);
    STD_TORCH_CHECK(b.size(1) == K, "a and b must have the same number of columns, got ", K, " and ", b.size(1));
    if (M <= 1) lda = (K + 15) / 16 * 16;
    if (N <= 1) ldb = (K + 15) / 16 * 16;
    STD_TORCH_CHECK(lda % 16 == 0 && ldb % 16 == 0 && is_aligned(a.const_data_ptr(), 16) &&
                        is_aligned(b.const_data_ptr(), 16),
                    "rows of a and b must start on 16-byte boundaries");
    const int64_t kb = blocks_of(K);
    STD_TORCH_CHECK(a_scale.scalar_type() == ST::Float && b_scale.scalar_type() == ST::Float, "scales must be float32");
    STD_TORCH_CHECK(a_scale.dim() == 2 && a_scale.size(0) == M && a_scale.size(1) == kb, "a_scale must be [", M, ", ", kb,
                    "]: one scale for each row and block of 128 columns of a");
    STD_TORCH_CHECK(b_scale.dim() == 2 && b_scale.size(1) == kb &&
                        (b_scale.size(0) == blocks_of(N) || b_scale.size(0) == N),
                    "b_scale must be [", blocks_of(N), ", ", kb, "], one scale for each 128 x 128 block of b, or [", N,
                    ", ", kb, "], one for each row and block of 128 columns");
    const bool by_row = b_scale.size(0) != blocks_of(N);
    a_scale = near_rows(a_scale);
    b_scale = near_rows(b_scale);
    const int64_t as_row = a_scale.size(0) > 1 ? a_scale.stride(0) : 0;
    const int64_t bs_row = b_scale.size(0) > 1 ? b_scale.stride(0) : 0;
    STD_TORCH_CHECK(out_type >= 0 && out_type <= 2, "the output must be bfloat16, float16 or float32");
    const int type = static_cast<int>(out_type);
    if (bias.has_value()) {
        STD_TORCH_CHECK(bias->is_cuda() && bias->get_device_index() == device_index, "bias must be on a's device");
        STD_TORCH_CHECK(value_type(*bias, "bias") == type, "bias must have the output's dtype");
        STD_TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N && (N <= 1 || bias->stride(0) == 1),
                        "bias must be a contiguous vector of N elements");
    }
    Tensor c = new_matrix(a, M, N, torch_dtype(type));
    if (M == 0 || N == 0) return c;
    const int64_t need = feather_block_scaled_mm_workspace_bytes(M, N, K);
    STD_TORCH_CHECK(need >= 0, "block_scaled_mm: sizes are out of range");
    if (need > 0) {
        STD_TORCH_CHECK(workspace.has_value() && workspace->is_cuda() && workspace->get_device_index() == device_index &&
                            workspace->scalar_type() == ST::Byte && workspace->is_contiguous() &&
                            workspace->numel() >= need && is_aligned(workspace->const_data_ptr(), 256),
                        "block_scaled_mm needs a contiguous uint8 workspace of at least ", need,
                        " bytes on a's device, 256-byte aligned");
    }
    torch::stable::accelerator::DeviceGuard guard(device_index);
    check_launch(feather_block_scaled_mm(
                     static_cast<const uint8_t*>(a.const_data_ptr()), lda, a_e5m2, floats(a_scale), as_row,
                     a_scale.stride(1), static_cast<const uint8_t*>(b.const_data_ptr()), ldb, b_e5m2, floats(b_scale), bs_row,
                     b_scale.stride(1), by_row, bias.has_value() ? bias->const_data_ptr() : nullptr,
                     c.mutable_data_ptr(), N, type, M, N, K, need > 0 ? workspace->mutable_data_ptr() : nullptr,
                     need > 0 ? workspace->numel() : 0, current_stream(device_index)),
                 "block_scaled_mm");
    return c;
}

// feather_ops::quantize_blocks (feather_quantize_blocks): codes [rows, cols], scale [rows, ceil(cols / 128)].
std::tuple<Tensor, Tensor> quantize_blocks(const Tensor& x, const bool e5m2) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int type = value_type(x, "x");
    const int64_t ldx = row_stride(x, "x");
    const int64_t rows = x.size(0);
    const int64_t cols = x.size(1);
    Codes q = new_codes(x, rows, cols, rows, e5m2);
    if (rows > 0 && cols > 0) {
        torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
        check_launch(feather_quantize_blocks(x.const_data_ptr(), type, ldx, bytes(q.codes), q.ld, floats(q.scale), 1,
                                             rows, e5m2, rows, cols, current_stream(x.get_device_index())),
                     "quantize_blocks");
    }
    return {q.codes, q.scale};
}

// feather_ops::quantize_tiles (feather_quantize_tiles): (codes, scale, codes of x^T, their scale, the column sums of each
// 128 rows), those asked for.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> quantize_tiles(const Tensor& x, const bool e5m2, const bool square,
                                                                  const bool plain, const bool transposed,
                                                                  const bool sums) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int type = value_type(x, "x");
    const int64_t ldx = row_stride(x, "x");
    const int64_t rows = x.size(0);
    const int64_t cols = x.size(1);
    STD_TORCH_CHECK(plain || transposed || sums, "nothing to compute");
    STD_TORCH_CHECK(rows > 0 && cols > 0, "x must not be empty");
    Codes q = plain ? new_codes(x, rows, cols, square ? blocks_of(rows) : rows, e5m2) : new_codes(x, 0, 0, 0, e5m2);
    Codes t = transposed ? new_codes(x, cols, rows, square ? blocks_of(cols) : cols, e5m2) : new_codes(x, 0, 0, 0, e5m2);
    Tensor s = sums ? new_matrix(x, blocks_of(rows), cols, aoti_torch_dtype_float32())
                    : new_matrix(x, 0, 0, aoti_torch_dtype_float32());
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    check_launch(feather_quantize_tiles(x.const_data_ptr(), type, ldx, square, plain ? bytes(q.codes) : nullptr, q.ld,
                                        plain ? floats(q.scale) : nullptr, 1, q.scale.size(0),
                                        transposed ? bytes(t.codes) : nullptr, t.ld,
                                        transposed ? floats(t.scale) : nullptr, 1, t.scale.size(0),
                                        sums ? floats(s) : nullptr, e5m2, rows, cols,
                                        current_stream(x.get_device_index())),
                 "quantize_tiles");
    return {q.codes, q.scale, t.codes, t.scale, s};
}

// feather_ops::sum_rows (feather_sum_rows): the column sums of a contiguous fp32 [rows, cols], in `out_type`.
Tensor sum_rows(const Tensor& part, const int64_t out_type) {
    STD_TORCH_CHECK(part.is_cuda() && part.scalar_type() == ST::Float && part.dim() == 2 && part.is_contiguous(),
                    "part must be a contiguous float32 CUDA matrix");
    STD_TORCH_CHECK(out_type >= 0 && out_type <= 2, "the output must be bfloat16, float16 or float32");
    STD_TORCH_CHECK(part.size(0) > 0 && part.size(1) > 0, "part must not be empty");
    Tensor out = new_vector(part, part.size(1), torch_dtype(static_cast<int>(out_type)));
    torch::stable::accelerator::DeviceGuard guard(part.get_device_index());
    check_launch(feather_sum_rows(floats(part), out.mutable_data_ptr(), static_cast<int>(out_type), part.size(0),
                                  part.size(1), current_stream(part.get_device_index())),
                 "sum_rows");
    return out;
}

struct NormArgs {
    int type;
    int64_t ldx, ld_residual, rows, cols;
    bool weight_fp32;
};

NormArgs check_norm(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int type = value_type(x, "x");
    const int64_t ldx = row_stride(x, "x");
    STD_TORCH_CHECK(x.size(0) > 0 && x.size(1) > 0, "x must not be empty");
    check_weight(weight, x);
    if (residual.has_value()) check_same(*residual, x, "residual");
    return {type, ldx, residual.has_value() ? row_stride(*residual, "residual") : 0, x.size(0), x.size(1),
            weight.scalar_type() == ST::Float};
}

// feather_ops::rms_norm (feather_rms_norm): (y, h = x + residual, 1 / rms of each row); h only with a residual, the last
// only where asked for.
std::tuple<Tensor, Tensor, Tensor> rms_norm(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual,
                                            const double eps, const bool need_rstd) {
    const NormArgs n = check_norm(x, weight, residual);
    const bool add = residual.has_value();
    Tensor y = new_matrix(x, n.rows, n.cols, torch_dtype(n.type));
    Tensor h = new_matrix(x, add ? n.rows : 0, add ? n.cols : 0, torch_dtype(n.type));
    Tensor rstd = new_vector(x, need_rstd ? n.rows : 0, aoti_torch_dtype_float32());
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    check_launch(feather_rms_norm(x.const_data_ptr(), n.ldx, add ? residual->const_data_ptr() : nullptr, n.ld_residual,
                                  weight.const_data_ptr(), n.weight_fp32, static_cast<float>(eps), n.type,
                                  add ? h.mutable_data_ptr() : nullptr, n.cols, y.mutable_data_ptr(), n.cols, nullptr, 0,
                                  nullptr, 0, 0, false, need_rstd ? floats(rstd) : nullptr, n.rows, n.cols,
                                  current_stream(x.get_device_index())),
                 "rms_norm");
    return {y, h, rstd};
}

// feather_ops::rms_norm_quantized: (codes, scale, h), h only with a residual.
std::tuple<Tensor, Tensor, Tensor> rms_norm_quantized(const Tensor& x, const Tensor& weight,
                                                      const std::optional<Tensor>& residual, const double eps,
                                                      const bool e5m2) {
    const NormArgs n = check_norm(x, weight, residual);
    const bool add = residual.has_value();
    Codes q = new_codes(x, n.rows, n.cols, n.rows, e5m2);
    Tensor h = new_matrix(x, add ? n.rows : 0, add ? n.cols : 0, torch_dtype(n.type));
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    check_launch(feather_rms_norm(x.const_data_ptr(), n.ldx, add ? residual->const_data_ptr() : nullptr, n.ld_residual,
                                  weight.const_data_ptr(), n.weight_fp32, static_cast<float>(eps), n.type,
                                  add ? h.mutable_data_ptr() : nullptr, n.cols, nullptr, 0, bytes(q.codes), q.ld,
                                  floats(q.scale), 1, n.rows, e5m2, nullptr, n.rows, n.cols,
                                  current_stream(x.get_device_index())),
                 "rms_norm_quantized");
    return {q.codes, q.scale, h};
}

// feather_ops::rms_norm_backward: (the gradient of x and of the residual, the weight's, in the weight's dtype).
std::tuple<Tensor, Tensor> rms_norm_backward(const Tensor& grad_y, const std::optional<Tensor>& grad_h, const Tensor& h,
                                             const Tensor& weight, const Tensor& rstd, const bool need_weight) {
    STD_TORCH_CHECK(h.is_cuda(), "h must be a CUDA tensor");
    const int type = value_type(h, "h");
    const int64_t ldh = row_stride(h, "h");
    const int64_t rows = h.size(0);
    const int64_t cols = h.size(1);
    STD_TORCH_CHECK(rows > 0 && cols > 0, "h must not be empty");
    check_same(grad_y, h, "grad_y");
    if (grad_h.has_value()) check_same(*grad_h, h, "grad_h");
    check_weight(weight, h);
    STD_TORCH_CHECK(rstd.is_cuda() && rstd.get_device_index() == h.get_device_index() &&
                        rstd.scalar_type() == ST::Float && rstd.dim() == 1 && rstd.size(0) == rows &&
                        rstd.is_contiguous(),
                    "rstd must be a contiguous float32 vector with one value for each row");
    Tensor grad_x = new_matrix(h, rows, cols, torch_dtype(type));
    const int64_t parts = feather_rms_norm_backward_parts(rows, cols);
    Tensor part = new_matrix(h, need_weight ? parts : 0, need_weight ? cols : 0, aoti_torch_dtype_float32());
    torch::stable::accelerator::DeviceGuard guard(h.get_device_index());
    const hipStream_t stream = current_stream(h.get_device_index());
    check_launch(feather_rms_norm_backward(grad_y.const_data_ptr(), row_stride(grad_y, "grad_y"),
                                           grad_h.has_value() ? grad_h->const_data_ptr() : nullptr,
                                           grad_h.has_value() ? row_stride(*grad_h, "grad_h") : 0, h.const_data_ptr(),
                                           ldh, weight.const_data_ptr(), weight.scalar_type() == ST::Float, floats(rstd),
                                           type, grad_x.mutable_data_ptr(), cols, need_weight ? floats(part) : nullptr,
                                           rows, cols, stream),
                 "rms_norm_backward");
    const int weight_type = value_type(weight, "weight");
    Tensor grad_w = new_vector(h, need_weight ? cols : 0, torch_dtype(weight_type));
    if (need_weight)
        check_launch(feather_sum_rows(floats(part), grad_w.mutable_data_ptr(), weight_type, parts, cols, stream),
                     "rms_norm_backward");
    return {grad_x, grad_w};
}

int64_t check_gate(const Tensor& x) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    STD_TORCH_CHECK(x.dim() == 2 && x.size(1) % 2 == 0, "x must have an even number of columns: the gate's and the "
                                                        "other factor's");
    STD_TORCH_CHECK(x.size(0) > 0 && x.size(1) > 0, "x must not be empty");
    return x.size(1) / 2;
}

// feather_ops::silu_mul (feather_silu_mul).
Tensor silu_mul(const Tensor& x) {
    const int64_t cols = check_gate(x);
    const int type = value_type(x, "x");
    Tensor y = new_matrix(x, x.size(0), cols, torch_dtype(type));
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    check_launch(feather_silu_mul(x.const_data_ptr(), row_stride(x, "x"), type, y.mutable_data_ptr(), cols, nullptr, 0,
                                  nullptr, 0, 0, false, x.size(0), cols, current_stream(x.get_device_index())),
                 "silu_mul");
    return y;
}

// feather_ops::silu_mul_quantized: (codes, scale).
std::tuple<Tensor, Tensor> silu_mul_quantized(const Tensor& x, const bool e5m2) {
    const int64_t cols = check_gate(x);
    const int type = value_type(x, "x");
    Codes q = new_codes(x, x.size(0), cols, x.size(0), e5m2);
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    check_launch(feather_silu_mul(x.const_data_ptr(), row_stride(x, "x"), type, nullptr, 0, bytes(q.codes), q.ld,
                                  floats(q.scale), 1, x.size(0), e5m2, x.size(0), cols,
                                  current_stream(x.get_device_index())),
                 "silu_mul_quantized");
    return {q.codes, q.scale};
}

// feather_ops::silu_mul_backward: x's gradient.
Tensor silu_mul_backward(const Tensor& grad_y, const Tensor& x) {
    const int64_t cols = check_gate(x);
    const int type = value_type(x, "x");
    STD_TORCH_CHECK(grad_y.is_cuda() && grad_y.get_device_index() == x.get_device_index() &&
                        grad_y.scalar_type() == x.scalar_type() && grad_y.dim() == 2 && grad_y.size(0) == x.size(0) &&
                        grad_y.size(1) == cols,
                    "grad_y must have the output's shape, x's dtype and device");
    Tensor grad_x = new_matrix(x, x.size(0), 2 * cols, torch_dtype(type));
    torch::stable::accelerator::DeviceGuard guard(x.get_device_index());
    check_launch(feather_silu_mul_backward(grad_y.const_data_ptr(), row_stride(grad_y, "grad_y"), x.const_data_ptr(),
                                           row_stride(x, "x"), type, grad_x.mutable_data_ptr(), 2 * cols, x.size(0), cols,
                                           current_stream(x.get_device_index())),
                 "silu_mul_backward");
    return grad_x;
}

}  // namespace

STABLE_TORCH_LIBRARY_FRAGMENT(feather_ops, m) {
    m.def(
        "block_scaled_mm(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, Tensor? bias, int out_type, "
        "Tensor(a!)? workspace) -> Tensor");
    m.def("quantize_blocks(Tensor x, bool e5m2) -> (Tensor, Tensor)");
    m.def(
        "quantize_tiles(Tensor x, bool e5m2, bool square, bool plain, bool transposed, bool sums) -> (Tensor, Tensor, "
        "Tensor, Tensor, Tensor)");
    m.def("sum_rows(Tensor part, int out_type) -> Tensor");
    m.def("rms_norm(Tensor x, Tensor weight, Tensor? residual, float eps, bool need_rstd) -> (Tensor, Tensor, Tensor)");
    m.def(
        "rms_norm_quantized(Tensor x, Tensor weight, Tensor? residual, float eps, bool e5m2) -> (Tensor, Tensor, "
        "Tensor)");
    m.def(
        "rms_norm_backward(Tensor grad_y, Tensor? grad_h, Tensor h, Tensor weight, Tensor rstd, bool need_weight) -> "
        "(Tensor, Tensor)");
    m.def("silu_mul(Tensor x) -> Tensor");
    m.def("silu_mul_quantized(Tensor x, bool e5m2) -> (Tensor, Tensor)");
    m.def("silu_mul_backward(Tensor grad_y, Tensor x) -> Tensor");
}

STABLE_TORCH_LIBRARY_IMPL(feather_ops, CUDA, m) {
    m.impl("block_scaled_mm", TORCH_BOX(&block_scaled_mm));
    m.impl("quantize_blocks", TORCH_BOX(&quantize_blocks));
    m.impl("quantize_tiles", TORCH_BOX(&quantize_tiles));
    m.impl("sum_rows", TORCH_BOX(&sum_rows));
    m.impl("rms_norm", TORCH_BOX(&rms_norm));
    m.impl("rms_norm_quantized", TORCH_BOX(&rms_norm_quantized));
    m.impl("rms_norm_backward", TORCH_BOX(&rms_norm_backward));
    m.impl("silu_mul", TORCH_BOX(&silu_mul));
    m.impl("silu_mul_quantized", TORCH_BOX(&silu_mul_quantized));
    m.impl("silu_mul_backward", TORCH_BOX(&silu_mul_backward));
}
