// Root-mean-square norm with the residual's addition, 16-bit, fp32 or block-scaled fp8 output, and its backward
// (include/feather_block_ops.h).
//
//   h = round(x + residual)     r = 1 / sqrt(sum(h^2) / cols + eps)     y = h r w
//   g = grad_y w, n = h r:      grad_h = r (g - n mean(g n)) + grad_h_in,   grad_w = sum over rows of grad_y n
//
// Both directions are streams through memory: a row is read once into registers (pieces of 8 values a lane), its sums
// are taken there, and what is written follows from the registers. Rows of up to 2048 values belong to one wave (sums
// by DPP, no barrier), longer ones to the four waves of a workgroup (one LDS exchange), and those past 16384 are read
// twice by one workgroup, the second time h as it was just written.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "block_common.h"

namespace feather {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct NormParams {
    const void* x;
    const void* residual;   // null: h = x
    const void* weight;
    void* h;
    void* y;                // null: q
    float* rstd;            // null: not kept
    Quantized q;
    int64_t ldx, ld_residual, ldh, ldy, rows;
    int32_t cols, weight_fp32;
    float eps;
};

struct NormBackwardParams {
    const void* grad_y;
    const void* grad_h_in;  // null: none
    const void* h;
    const void* weight;
    const float* rstd;
    void* grad_h;
    float* part;            // null: no weight gradient
    int64_t ld_grad_y, ld_grad_h_in, ldh, ld_grad_h, rows;
    int32_t cols, weight_fp32;
};

template <int kType>
__device__ __forceinline__ const void* row_at(const void* p, int64_t row, int64_t ld) {
    return static_cast<const uint8_t*>(p) + row * ld * type_bytes(kType);
}

template <int kType>
__device__ __forceinline__ void* row_at(void* p, int64_t row, int64_t ld) {
    return static_cast<uint8_t*>(p) + row * ld * type_bytes(kType);
}

// The sum over the kRowWaves waves that share a row, in all of their lanes.
template <int kRowWaves>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    v = sum64(v);
    if constexpr (kRowWaves > 1) {
        static_assert(kRowWaves == kWaves, "a row has one wave or the whole workgroup");
        __syncthreads();   // the last exchange's values have been read
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
        __syncthreads();
        v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    }
    return v;
}

// x + residual rounded to the type, kept as h (or x alone).
template <int kType, bool kVec>
__device__ __forceinline__ void stream_piece(const NormParams& p, int64_t row, int at, int valid, float (&v)[kPiece]) {
    load_piece<kType, kVec>(row_at<kType>(p.x, row, p.ldx), at, valid, v);
    if (p.residual) {
        float res[kPiece];
        load_piece<kType, kVec>(row_at<kType>(p.residual, row, p.ld_residual), at, valid, res);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) v[i] = to_float<kType>(to_bits<kType>(v[i] + res[i]));
        store_piece<kType, kVec>(row_at<kType>(p.h, row, p.ldh), at, valid, v);
    }
}

template <int kType, bool kVec>
__device__ __forceinline__ void write_piece(const NormParams& p, int64_t row, int at, int valid, float r,
                                            float (&v)[kPiece]) {
    float w[kPiece];
    load_weight<kType, kVec>(p.weight, p.weight_fp32, at, valid, w);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) v[i] = v[i] * r * w[i];
    if (p.y) store_piece<kType, kVec>(row_at<kType>(p.y, row, p.ldy), at, valid, v);
    else quantize_piece<kVec>(p.q, row, at, valid, v);
}

// kPieces: pieces per lane, all of the row's in registers (0: a row of any length, read twice).
template <int kType, bool kVec, int kRowWaves, int kPieces>
__global__ __launch_bounds__(kThreads) void norm_kernel(const NormParams p) {
    constexpr int kRowThreads = 64 * kRowWaves;
    __shared__ float lds[kWaves];
    const int t = threadIdx.x % kRowThreads;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / kRowThreads) + threadIdx.x / kRowThreads;
    if (row >= p.rows) return;   // whole waves, and only where a row is a wave's own: no barrier is missed
    float sum = 0.0f;
    if constexpr (kPieces > 0) {
        float v[kPieces][kPiece];
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            stream_piece<kType, kVec>(p, row, at, p.cols - at, v[c]);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) sum += v[c][i] * v[c][i];
        }
        const float r = 1.0f / sqrtf(row_sum<kRowWaves>(sum, lds) / static_cast<float>(p.cols) + p.eps);
        if (t == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            write_piece<kType, kVec>(p, row, at, p.cols - at, r, v[c]);
        }
    } else {
        const int steps = (p.cols + kRowThreads * kPiece - 1) / (kRowThreads * kPiece);
        for (int c = 0; c < steps; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            float v[kPiece];
            stream_piece<kType, kVec>(p, row, at, p.cols - at, v);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) sum += v[i] * v[i];
        }
        const float r = 1.0f / sqrtf(row_sum<kRowWaves>(sum, lds) / static_cast<float>(p.cols) + p.eps);
        if (t == 0 && p.rstd) p.rstd[row] = r;
        const void* from = p.residual ? row_at<kType>(static_cast<const void*>(p.h), row, p.ldh)
                                      : row_at<kType>(p.x, row, p.ldx);
        for (int c = 0; c < steps; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            float v[kPiece];
            load_piece<kType, kVec>(from, at, p.cols - at, v);   // what this lane itself wrote
            write_piece<kType, kVec>(p, row, at, p.cols - at, r, v);
        }
    }
}

// One piece of grad_h.
template <int kType, bool kVec>
__device__ __forceinline__ void write_grad(const NormBackwardParams& p, int64_t row, int at, int valid, float r,
                                           float mean, const float (&g)[kPiece], const float (&n)[kPiece]) {
    float out[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece; ++i) out[i] = r * (g[i] - n[i] * mean);
    if (p.grad_h_in) {
        float in[kPiece];
        load_piece<kType, kVec>(row_at<kType>(p.grad_h_in, row, p.ld_grad_h_in), at, valid, in);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) out[i] += in[i];
    }
    store_piece<kType, kVec>(row_at<kType>(p.grad_h, row, p.ld_grad_h), at, valid, out);
}

// Rows blockIdx.x * R + (which of the workgroup's), and every gridDim.x * R on: the lanes keep the sums of grad_y n of
// their columns over all of them.
template <int kType, bool kVec, int kRowWaves, int kPieces>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(const NormBackwardParams p) {
    constexpr int kRowThreads = 64 * kRowWaves;
    constexpr int kRows = kThreads / kRowThreads;
    __shared__ float lds[kRowWaves > 1 ? kWaves : kWaves * 64 * kPiece];
    const int t = threadIdx.x % kRowThreads;
    float dw[kPieces][kPiece] = {};
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kRowThreads; row < p.rows;
         row += static_cast<int64_t>(gridDim.x) * kRows) {
        const float r = p.rstd[row];
        float g[kPieces][kPiece], n[kPieces][kPiece], sum = 0.0f;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece, valid = p.cols - at;
            float w[kPiece];
            load_piece<kType, kVec>(row_at<kType>(p.grad_y, row, p.ld_grad_y), at, valid, g[c]);
            load_piece<kType, kVec>(row_at<kType>(p.h, row, p.ldh), at, valid, n[c]);
            load_weight<kType, kVec>(p.weight, p.weight_fp32, at, valid, w);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                n[c][i] *= r;
                dw[c][i] += g[c][i] * n[c][i];
                g[c][i] *= w[i];
                sum += g[c][i] * n[c][i];
            }
        }
        const float mean = row_sum<kRowWaves>(sum, lds) / static_cast<float>(p.cols);
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            write_grad<kType, kVec>(p, row, at, p.cols - at, r, mean, g[c], n[c]);
        }
    }
    if (!p.part) return;
    float* part = p.part + static_cast<int64_t>(blockIdx.x) * p.cols;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
        const int at = (c * kRowThreads + t) * kPiece;
        if constexpr (kRowWaves == 1) {   // the four waves' rows: joined in wave order
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPiece; ++i) lds[(i * kWaves + threadIdx.x / 64) * 64 + t] = dw[c][i];
            __syncthreads();
            if (threadIdx.x >= 64) continue;
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) s += lds[(i * kWaves + w) * 64 + t];
                dw[c][i] = s;
            }
        }
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
            if (at + i < p.cols) part[at + i] = dw[c][i];
    }
}

// Rows past 16384 values: grad_h alone, two readings; the weight's sums are long_weight_kernel's.
template <int kType, bool kVec>
__global__ __launch_bounds__(kThreads) void norm_backward_long_kernel(const NormBackwardParams p) {
    __shared__ float lds[kWaves];
    const int64_t row = blockIdx.x;
    const int steps = (p.cols + kThreads * kPiece - 1) / (kThreads * kPiece);
    const float r = p.rstd[row];
    float sum = 0.0f, mean = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
        for (int c = 0; c < steps; ++c) {
            const int at = (c * kThreads + static_cast<int>(threadIdx.x)) * kPiece, valid = p.cols - at;
            float g[kPiece], n[kPiece], w[kPiece];
            load_piece<kType, kVec>(row_at<kType>(p.grad_y, row, p.ld_grad_y), at, valid, g);
            load_piece<kType, kVec>(row_at<kType>(p.h, row, p.ldh), at, valid, n);
            load_weight<kType, kVec>(p.weight, p.weight_fp32, at, valid, w);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                n[i] *= r;
                g[i] *= w[i];
                sum += g[i] * n[i];
            }
            if (pass == 1) write_grad<kType, kVec>(p, row, at, valid, r, mean, g, n);
        }
        if (pass == 0) mean = row_sum<kWaves>(sum, lds) / static_cast<float>(p.cols);
    }
}

// The weight's sums over rows blockIdx.y, + gridDim.y, ... of the columns of workgroup column blockIdx.x.
template <int kType, bool kVec>
__global__ __launch_bounds__(kThreads) void long_weight_kernel(const NormBackwardParams p) {
    const int at = (static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x)) * kPiece;
    const int valid = p.cols - at;
    if (valid <= 0) return;
    float dw[kPiece] = {};
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        float g[kPiece], n[kPiece];
        load_piece<kType, kVec>(row_at<kType>(p.grad_y, row, p.ld_grad_y), at, valid, g);
        load_piece<kType, kVec>(row_at<kType>(p.h, row, p.ldh), at, valid, n);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) dw[i] += g[i] * (n[i] * p.rstd[row]);
    }
    float* part = p.part + static_cast<int64_t>(blockIdx.y) * p.cols;
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
        if (i < valid) part[at + i] = dw[i];
}

// out[j] = the sum of part[., j]: a workgroup takes 64 columns, its waves every fourth row each, joined in wave order.
template <int kType>
__global__ __launch_bounds__(kThreads) void sum_rows_kernel(const float* part, void* out, int64_t rows, int64_t cols) {
    __shared__ float lds[kThreads];
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x % 64;
    float s = 0.0f;
    if (col < cols)
        for (int64_t i = threadIdx.x / 64; i < rows; i += kWaves) s += part[i * cols + col];
    lds[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x >= 64 || col >= cols) return;
    s = (lds[threadIdx.x] + lds[threadIdx.x + 64]) + (lds[threadIdx.x + 128] + lds[threadIdx.x + 192]);
    if constexpr (kType == FEATHER_FP32) static_cast<uint32_t*>(out)[col] = to_bits<kType>(s);
    else static_cast<uint16_t*>(out)[col] = static_cast<uint16_t>(to_bits<kType>(s));
}

constexpr int64_t kMaxGrid = (int64_t{1} << 31) - 1;
constexpr int64_t kWaveCols = 2048;       // rows up to here are one wave's
constexpr int64_t kRegisterCols = 16384;  // and up to here in registers
constexpr int64_t kLongParts = 64;

// Workgroups of the backward: 512 (two a CU), fewer where the rows are.
int64_t backward_groups(int64_t rows, int64_t cols) {
    if (cols > kRegisterCols) return rows < kLongParts ? rows : kLongParts;
    const int64_t groups = cols <= kWaveCols ? (rows + kWaves - 1) / kWaves : rows;
    return groups < 512 ? groups : 512;
}

// Calls f<type, vec>() for the runtime values.
template <typename F>
void by_type(int type, bool vec, F&& f) {
    const auto go = [&](auto t) {
        if (vec) f(t, std::true_type{});
        else f(t, std::false_type{});
    };
    if (type == FEATHER_BF16) go(std::integral_constant<int, FEATHER_BF16>{});
    else if (type == FEATHER_FP16) go(std::integral_constant<int, FEATHER_FP16>{});
    else go(std::integral_constant<int, FEATHER_FP32>{});
}

// Calls f<waves per row, pieces per lane>() for rows of `cols` values (at most kRegisterCols).
template <typename F>
void by_cols(int64_t cols, F&& f) {
    const auto go = [&](auto waves, auto pieces) { f(waves, pieces); };
    using W1 = std::integral_constant<int, 1>;
    using W4 = std::integral_constant<int, kWaves>;
    if (cols <= 512) go(W1{}, std::integral_constant<int, 1>{});
    else if (cols <= 1024) go(W1{}, std::integral_constant<int, 2>{});
    else if (cols <= 2048) go(W1{}, std::integral_constant<int, 4>{});
    else if (cols <= 4096) go(W4{}, std::integral_constant<int, 2>{});
    else if (cols <= 6144) go(W4{}, std::integral_constant<int, 3>{});
    else if (cols <= 8192) go(W4{}, std::integral_constant<int, 4>{});
    else go(W4{}, std::integral_constant<int, 8>{});
}

bool weight_on_16(const void* weight) { return on_16(weight); }

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" bool feather_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ld_residual,
                                 const void* weight, bool weight_fp32, float eps, int type, void* h, int64_t ldh,
                                 void* y, int64_t ldy, uint8_t* codes, int64_t ld_codes, float* scale,
                                 int64_t scale_row, int64_t scale_block, bool e5m2, float* rstd, int64_t rows,
                                 int64_t cols, hipStream_t stream) {
    if (!type_ok(type) || !matrix_ok(x, ldx, rows, cols) || !weight) return false;
    const int weight_type = weight_fp32 ? static_cast<int>(FEATHER_FP32) : type;
    if (!aligned_to_type(x, type) || !aligned_to_type(weight, weight_type)) return false;
    if ((residual == nullptr) != (h == nullptr)) return false;
    if (residual && (!matrix_ok(residual, ld_residual, rows, cols) || !matrix_ok(h, ldh, rows, cols) ||
                     !aligned_to_type(residual, type) || !aligned_to_type(h, type)))
        return false;
    if (y ? codes || scale || !matrix_ok(y, ldy, rows, cols) || !aligned_to_type(y, type)
          : !quantized_ok(codes, ld_codes, scale, rows, cols))
        return false;
    const NormParams p{x, residual, weight, h, y, rstd, {codes, scale, ld_codes, scale_row, scale_block, e5m2},
                       ldx, ld_residual, ldh, ldy, rows, static_cast<int32_t>(cols), weight_fp32, eps};
    const bool vec = rows_on_16(x, ldx, type) && weight_on_16(weight) &&
                     (!residual || (rows_on_16(residual, ld_residual, type) && rows_on_16(h, ldh, type))) &&
                     (y ? rows_on_16(y, ldy, type) : (on_16(codes) && ld_codes % 8 == 0));
    const int64_t groups = cols <= kWaveCols ? (rows + kWaves - 1) / kWaves : rows;
    if (groups > kMaxGrid) return false;
    by_type(type, vec, [&](auto t, auto v) {
        if (cols > kRegisterCols) {
            norm_kernel<t(), v(), kWaves, 0><<<static_cast<uint32_t>(groups), kThreads, 0, stream>>>(p);
            return;
        }
        by_cols(cols, [&](auto waves, auto pieces) {
            norm_kernel<t(), v(), waves(), pieces()><<<static_cast<uint32_t>(groups), kThreads, 0, stream>>>(p);
        });
    });
    return true;
}

extern "C" int64_t feather_rms_norm_backward_parts(int64_t rows, int64_t cols) {
    return rows >= 1 && cols >= 1 ? backward_groups(rows, cols) : 0;
}

extern "C" bool feather_rms_norm_backward(const void* grad_y, int64_t ld_grad_y, const void* grad_h_in,
                                          int64_t ld_grad_h_in, const void* h, int64_t ldh, const void* weight,
                                          bool weight_fp32, const float* rstd, int type, void* grad_h,
                                          int64_t ld_grad_h, float* part, int64_t rows, int64_t cols,
                                          hipStream_t stream) {
    if (!type_ok(type) || !matrix_ok(grad_y, ld_grad_y, rows, cols) || !matrix_ok(h, ldh, rows, cols) ||
        !matrix_ok(grad_h, ld_grad_h, rows, cols) || !weight || !rstd)
        return false;
    if (grad_h_in && (!matrix_ok(grad_h_in, ld_grad_h_in, rows, cols) || !aligned_to_type(grad_h_in, type))) return false;
    const int weight_type = weight_fp32 ? static_cast<int>(FEATHER_FP32) : type;
    if (!aligned_to_type(grad_y, type) || !aligned_to_type(h, type) || !aligned_to_type(grad_h, type) ||
        !aligned_to_type(weight, weight_type))
        return false;
    const NormBackwardParams p{grad_y, grad_h_in, h, weight, rstd, grad_h, part, ld_grad_y, ld_grad_h_in, ldh,
                               ld_grad_h, rows, static_cast<int32_t>(cols), weight_fp32};
    const bool vec = rows_on_16(grad_y, ld_grad_y, type) && rows_on_16(h, ldh, type) &&
                     rows_on_16(grad_h, ld_grad_h, type) && weight_on_16(weight) &&
                     (!grad_h_in || rows_on_16(grad_h_in, ld_grad_h_in, type));
    const auto groups = static_cast<uint32_t>(backward_groups(rows, cols));
    by_type(type, vec, [&](auto t, auto v) {
        if (cols > kRegisterCols) {
            norm_backward_long_kernel<t(), v()><<<static_cast<uint32_t>(rows), kThreads, 0, stream>>>(p);
            if (!part) return;
            const auto strips = static_cast<uint32_t>((cols + kThreads * kPiece - 1) / (kThreads * kPiece));
            long_weight_kernel<t(), v()><<<dim3(strips, groups), kThreads, 0, stream>>>(p);
            return;
        }
        by_cols(cols, [&](auto waves, auto pieces) {
            norm_backward_kernel<t(), v(), waves(), pieces()><<<groups, kThreads, 0, stream>>>(p);
        });
    });
    return true;
}

extern "C" bool feather_sum_rows(const float* part, void* out, int type, int64_t rows, int64_t cols,
                                 hipStream_t stream) {
    if (!part || !out || !type_ok(type) || rows < 1 || cols < 1 || !aligned_to_type(out, type)) return false;
    const int64_t groups = (cols + 63) / 64;
    if (groups > kMaxGrid) return false;
    by_type(type, true, [&](auto t, auto) {
        sum_rows_kernel<t()><<<static_cast<uint32_t>(groups), kThreads, 0, stream>>>(part, out, rows, cols);
    });
    return true;
}
