// Gated activation silu(gate) * up with 16-bit, fp32 or block-scaled fp8 output, its backward, and the quantization of
// rows to blocks of 128 (include/feather_block_ops.h).
//
//   s = 1 / (1 + exp(-g))     y = g s u     grad_u = grad_y g s     grad_g = grad_y u s (1 + g (1 - s))
//
// Streams through memory: a lane takes one piece of 8 values at a time, the 16 lanes of a block together. Pieces are
// counted over all rows, whole blocks to a row, so that short rows fill the waves too. Memory bounds it: fp8 from fp16 4096 x
// 12288 45.3 us, 5.6 TB/s; gradients of bf16 1000 x 13824 21.9, 6.3 (138 MB, less than the last-level cache); 16 rows 3.2, a launch's time.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "block_common.h"

namespace feather {
namespace {

constexpr int kThreads = 256;

enum class Op { kQuantize, kSiluMul, kSiluMulBackward };

struct RowsParams {
    const void* x;          // the values; gate and up side by side
    const void* grad_y;
    void* y;                // null: q; grad_x of the backward
    Quantized q;
    int64_t ldx, ld_grad_y, ldy, rows;
    int32_t cols, pieces;   // of a row: a multiple of 16
};

template <int kType>
__device__ __forceinline__ const void* row_at(const void* p, int64_t row, int64_t ld) {
    return static_cast<const uint8_t*>(p) + row * ld * type_bytes(kType);
}

// s = 1 / (1 + exp(-g)) and half of c = 1 - s. With t = exp(-|g|) and q = 1 / (1 + t) they are q and t q, or the other way round. NaN
// stays NaN. fp32: the exponential within an ulp, a true division, and c as a product, which keeps its bits where s is near 1;
// 7 roundings in all for g s (by the other types' instructions up to 80 where |g| is 80), in the same time (4096 x 12288 102
// us; to fp8 85.5 against 84). 16-bit types, whose own rounding hides those (4096 x 12288 fp16 to fp8 fp32's way: 64 us for 43,
// codes other than the 64-bit definition's 64 for 77 of 100 million, by plain 32-bit operations 84): the exponential instruction, whose argument's
// rounding costs |g| 2^-24 of t, squared so that it reaches below the least normal without losing its bits; q's argument is
// in [1, 2], where the reciprocal instruction (1 ulp) needs none of a division's scaling; c as a difference (as a product
// the backward of 13.8 million gradients in cache took 22.3 us, not 21.8).
struct Sigmoid {
    float s, half_c;
};

template <int kType>
__device__ __forceinline__ Sigmoid sigmoid(float g) {
    if constexpr (kType == FEATHER_FP32) {
        const float t = expf(-fabsf(g));
        const float q = 1.0f / (1.0f + t);
        const float tq = t * q;
        return g < 0.0f ? Sigmoid{tq, 0.5f * q} : Sigmoid{q, 0.5f * tq};
    } else {
        const float root = __expf(-0.5f * fabsf(g));
        const float t = root * root;
        const float q = __builtin_amdgcn_rcpf(1.0f + t);
        const float s = g < 0.0f ? t * q : q;
        return {s, 0.5f - 0.5f * s};
    }
}

// a b c for |c| <= 1 without a step that leaves the range where the product does not: the larger of a and b takes c.
__device__ __forceinline__ float product(float a, float b, float c) {
    const bool first = fabsf(a) > fabsf(b);
    return (first ? a : b) * c * (first ? b : a);
}

template <Op kOp, int kType, bool kVec>
__global__ __launch_bounds__(kThreads) void rows_kernel(const RowsParams p) {
    // The workgroup's first piece as (row, piece of it), then this lane's from there in 32 bits.
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads;
    const int64_t first_row = first / p.pieces;
    const uint32_t piece0 = static_cast<uint32_t>(first - first_row * p.pieces) + threadIdx.x;
    const uint32_t more = piece0 / static_cast<uint32_t>(p.pieces);
    const int64_t row = first_row + more;
    if (row >= p.rows) return;   // whole blocks of lanes: a row's pieces are a multiple of 16
    const int at = static_cast<int>(piece0 - more * static_cast<uint32_t>(p.pieces)) * kPiece;
    const int valid = p.cols - at;
    float v[kPiece];
    const void* x = row_at<kType>(p.x, row, p.ldx);
    load_piece<kType, kVec>(x, at, valid, v);
    if constexpr (kOp != Op::kQuantize) {
        float up[kPiece];
        load_piece<kType, kVec>(x, p.cols + at, valid, up);
        if constexpr (kOp == Op::kSiluMul) {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) v[i] = v[i] * sigmoid<kType>(v[i]).s * up[i];
        } else {
            float g[kPiece];
            load_piece<kType, kVec>(row_at<kType>(p.grad_y, row, p.ld_grad_y), at, valid, g);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                const auto [s, half_c] = sigmoid<kType>(v[i]);
                // v s first: of a gate masked with the type's lowest value it is 0, and grad_y v may be infinite. 13.8 million
                // gradients in cache, 21.5 us with products from the left, take 21.8 so.
                const float grad_up = g[i] * (v[i] * s);
                v[i] = 2.0f * product(g[i], up[i], s * (0.5f + v[i] * half_c));   // silu's slope is at most 1.1
                up[i] = grad_up;
            }
            void* out = static_cast<uint8_t*>(p.y) + row * p.ldy * type_bytes(kType);
            store_piece<kType, kVec>(out, at, valid, v);
            store_piece<kType, kVec>(out, p.cols + at, valid, up);
            return;
        }
        if (p.y) {
            store_piece<kType, kVec>(static_cast<uint8_t*>(p.y) + row * p.ldy * type_bytes(kType), at, valid, v);
            return;
        }
    }
    quantize_piece<kVec, std::conditional_t<kOp == Op::kQuantize, ExactFactor, Factor>>(p.q, row, at, valid, v);
}

// p from row `row` on.
RowsParams from_row(RowsParams p, int64_t row, int type) {
    const int bytes = type_bytes(type);
    p.x = static_cast<const uint8_t*>(p.x) + row * p.ldx * bytes;
    if (p.grad_y) p.grad_y = static_cast<const uint8_t*>(p.grad_y) + row * p.ld_grad_y * bytes;
    if (p.y) p.y = static_cast<uint8_t*>(p.y) + row * p.ldy * bytes;
    p.q = from_row(p.q, row);
    p.rows -= row;
    return p;
}

template <Op kOp>
bool launch(const RowsParams& p, int type, bool vec, hipStream_t stream) {
    const int64_t most = (kMaxThreads - kThreads) / p.pieces;   // rows of a launch, a lane to each piece
    const auto go = [&](auto t) {
        for (int64_t row = 0; row < p.rows; row += most) {
            RowsParams part = from_row(p, row, type);
            part.rows = std::min(part.rows, most);
            const auto groups = static_cast<uint32_t>((part.rows * p.pieces + kThreads - 1) / kThreads);
            if (vec) rows_kernel<kOp, t(), true><<<groups, kThreads, 0, stream>>>(part);
            else rows_kernel<kOp, t(), false><<<groups, kThreads, 0, stream>>>(part);
        }
    };
    if (type == FEATHER_BF16) go(std::integral_constant<int, FEATHER_BF16>{});
    else if (type == FEATHER_FP16) go(std::integral_constant<int, FEATHER_FP16>{});
    else go(std::integral_constant<int, FEATHER_FP32>{});
    return true;
}

int32_t pieces_of(int64_t cols) { return static_cast<int32_t>((cols + kBlock - 1) / kBlock * (kBlock / kPiece)); }

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" bool feather_quantize_blocks(const void* x, int type, int64_t ldx, uint8_t* codes, int64_t ld_codes,
                                        float* scale, int64_t scale_row, int64_t scale_block, bool e5m2, int64_t rows,
                                        int64_t cols, hipStream_t stream) {
    if (!type_ok(type) || !matrix_ok(x, ldx, rows, cols) || !aligned_to_type(x, type) ||
        !quantized_ok(codes, ld_codes, scale, rows, cols))
        return false;
    const RowsParams p{x, nullptr, nullptr, {codes, scale, ld_codes, scale_row, scale_block, e5m2}, ldx, 0, 0, rows,
                       static_cast<int32_t>(cols), pieces_of(cols)};
    return launch<Op::kQuantize>(
        p, type, cols % kPiece == 0 && rows_on_16(x, ldx, type) && on_16(codes) && ld_codes % 8 == 0, stream);
}

extern "C" bool feather_silu_mul(const void* x, int64_t ldx, int type, void* y, int64_t ldy, uint8_t* codes,
                                 int64_t ld_codes, float* scale, int64_t scale_row, int64_t scale_block, bool e5m2,
                                 int64_t rows, int64_t cols, hipStream_t stream) {
    if (!type_ok(type) || !matrix_ok(x, ldx, rows, cols) || ldx < 2 * cols || !aligned_to_type(x, type)) return false;
    if (y ? codes || scale || !matrix_ok(y, ldy, rows, cols) || !aligned_to_type(y, type)
          : !quantized_ok(codes, ld_codes, scale, rows, cols))
        return false;
    const RowsParams p{x, nullptr, y, {codes, scale, ld_codes, scale_row, scale_block, e5m2}, ldx, 0, ldy, rows,
                       static_cast<int32_t>(cols), pieces_of(cols)};
    // whole pieces; then up, which starts at column cols, is on a 16-byte boundary too
    const bool vec = cols % kPiece == 0 && rows_on_16(x, ldx, type) &&
                     (y ? rows_on_16(y, ldy, type) : (on_16(codes) && ld_codes % 8 == 0));
    return launch<Op::kSiluMul>(p, type, vec, stream);
}

extern "C" bool feather_silu_mul_backward(const void* grad_y, int64_t ld_grad_y, const void* x, int64_t ldx, int type,
                                          void* grad_x, int64_t ld_grad_x, int64_t rows, int64_t cols,
                                          hipStream_t stream) {
    if (!type_ok(type) || !matrix_ok(x, ldx, rows, cols) || ldx < 2 * cols || !matrix_ok(grad_y, ld_grad_y, rows, cols) ||
        !matrix_ok(grad_x, ld_grad_x, rows, cols) || ld_grad_x < 2 * cols || !aligned_to_type(x, type) ||
        !aligned_to_type(grad_y, type) || !aligned_to_type(grad_x, type))
        return false;
    const RowsParams p{x, grad_y, grad_x, {}, ldx, ld_grad_y, ld_grad_x, rows, static_cast<int32_t>(cols),
                       pieces_of(cols)};
    const bool vec = cols % kPiece == 0 && rows_on_16(x, ldx, type) &&
                     rows_on_16(grad_y, ld_grad_y, type) && rows_on_16(grad_x, ld_grad_x, type);
    return launch<Op::kSiluMulBackward>(p, type, vec, stream);
}
