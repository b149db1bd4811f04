// Root-mean-square norm with the residual's addition, 16-bit, fp32 or block-scaled fp8 output, and its backward
// (include/feather_block_ops.h).
//
//   h = round(x + residual)     r = 1 / sqrt(sum(h^2) / cols + eps)     y = h r w
//   g = grad_y w, n = h r:      grad_h = r (g - n mean(g n)) + grad_h_in,   grad_w = sum over rows of grad_y n
//
// Both directions are streams through memory: a row is read once into registers (pieces of 8 values a lane), its sums
// are taken there, and what is written follows from the registers. Rows of up to 2048 values belong to one wave (sums
// by DPP, no barrier), longer ones to the four to sixteen waves of a workgroup (one LDS exchange; sixteen where there are no
// more rows than CUs: one row of 14336 9.6 -> 5.5 us), and those past 16384 are read twice by one workgroup, the second time h
// as it was just written.
//
// Measured against a copy's 4.96 TB/s (read and written): forward with fp8 output 4112 x 5120 fp16 28.6 us, 5.1 TB/s; backward
// of 4096 x 4096 bf16 25 us, 5.4 TB/s, and 4 us for the weight's sums; one row of 4096 2.9 us, a launch's time.
#include <hip/hip_runtime.h>

#include <algorithm>
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

// Threads of a workgroup whose rows have kRowWaves waves each.
constexpr int threads_of(int row_waves) { return row_waves > kWaves ? 64 * row_waves : kThreads; }

// The sum over the kRowWaves waves that share a row, in all of their lanes.
template <int kRowWaves>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    v = sum64(v);
    if constexpr (kRowWaves > 1) {
        static_assert(64 * kRowWaves == threads_of(kRowWaves), "a row has one wave or the whole workgroup");
        __syncthreads();   // the last exchange's values have been read
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w) v += lds[w];
    }
    return v;
}

// x + residual rounded to the type, kept as h (or x alone).
template <int kType, bool kVec>
__device__ __forceinline__ void stream_piece(const NormParams& p, int64_t row, int at, int valid, const RawPiece<kType>& x,
                                             const RawPiece<kType>& residual, float (&v)[kPiece]) {
    unpack(x, v);
    if (p.residual) {
        float res[kPiece];
        unpack(residual, res);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) v[i] = to_float<kType>(to_bits<kType>(v[i] + res[i]));
        if (valid > 0) store_piece<kType, kVec>(row_at<kType>(p.h, row, p.ldh), at, valid, v);
    }
}

// y = v r w, and where it goes. raw_w: the weight's piece where it has the activations' type.
template <int kType, bool kVec>
__device__ __forceinline__ void write_piece(const NormParams& p, int64_t row, int at, int valid, float r,
                                            float (&v)[kPiece], const RawPiece<kType>& raw_w) {
    float w[kPiece];
    if (p.weight_fp32) load_piece<FEATHER_FP32, kVec>(p.weight, at, valid, w);
    else unpack(raw_w, w);
    if (p.y) {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) v[i] = v[i] * r * w[i];
        if (valid > 0) store_piece<kType, kVec>(row_at<kType>(p.y, row, p.ldy), at, valid, v);
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) v[i] *= w[i];
        quantize_piece<kVec, RowFactor>(p.q, row, at, valid, v, r);
    }
}

template <int kType, bool kVec>
__device__ __forceinline__ RawPiece<kType> weight_piece(const void* weight, bool fp32, int at, int valid) {
    return fp32 ? RawPiece<kType>{} : load_raw<kType, kVec>(weight, at, valid);
}

// kPieces: pieces per lane, all of the row's in registers (0: a row of any length, read twice).
template <int kType, bool kVec, int kRowWaves, int kPieces>
__global__ __launch_bounds__(threads_of(kRowWaves)) void norm_kernel(const NormParams p) {
    constexpr int kRowThreads = 64 * kRowWaves;
    constexpr int kRows = threads_of(kRowWaves) / kRowThreads;
    __shared__ float lds[kRowWaves > 1 ? kRowWaves : 1];
    const int t = threadIdx.x % kRowThreads;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kRowThreads;
    if (row >= p.rows) return;   // whole waves, and only where a row is a wave's own: no barrier is missed
    float sum = 0.0f;
    if constexpr (kPieces > 0) {
        RawPiece<kType> x[kPieces], res[kPieces], w[kPieces];   // all loads ahead of the first use
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            x[c] = load_raw<kType, kVec>(row_at<kType>(p.x, row, p.ldx), at, p.cols - at);
        }
        if (p.residual) {
#pragma unroll
            for (int c = 0; c < kPieces; ++c) {
                const int at = (c * kRowThreads + t) * kPiece;
                res[c] = load_raw<kType, kVec>(row_at<kType>(p.residual, row, p.ld_residual), at, p.cols - at);
            }
        }
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            w[c] = weight_piece<kType, kVec>(p.weight, p.weight_fp32, at, p.cols - at);
        }
        float v[kPieces][kPiece];
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            stream_piece<kType, kVec>(p, row, at, p.cols - at, x[c], res[c], v[c]);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) sum += v[c][i] * v[c][i];
        }
        const float r = 1.0f / sqrtf(row_sum<kRowWaves>(sum, lds) / static_cast<float>(p.cols) + p.eps);
        if (t == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            write_piece<kType, kVec>(p, row, at, p.cols - at, r, v[c], w[c]);
        }
    } else {
        const int steps = (p.cols + kRowThreads * kPiece - 1) / (kRowThreads * kPiece);
        for (int c = 0; c < steps; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            float v[kPiece];
            const RawPiece<kType> x = load_raw<kType, kVec>(row_at<kType>(p.x, row, p.ldx), at, p.cols - at);
            RawPiece<kType> res{};
            if (p.residual)
                res = load_raw<kType, kVec>(row_at<kType>(p.residual, row, p.ld_residual), at, p.cols - at);
            stream_piece<kType, kVec>(p, row, at, p.cols - at, x, res, v);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) sum += v[i] * v[i];
        }
        const float r = 1.0f / sqrtf(row_sum<kRowWaves>(sum, lds) / static_cast<float>(p.cols) + p.eps);
        if (t == 0 && p.rstd) p.rstd[row] = r;
        // What a lane reads of h it wrote itself; a lane past the row's end reads the first piece and drops it.
        const void* from = p.residual ? row_at<kType>(static_cast<const void*>(p.h), row, p.ldh)
                                      : row_at<kType>(p.x, row, p.ldx);
        for (int c = 0; c < steps; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            float v[kPiece];
            load_piece<kType, kVec>(from, at, p.cols - at, v);
            write_piece<kType, kVec>(p, row, at, p.cols - at, r, v,
                                     weight_piece<kType, kVec>(p.weight, p.weight_fp32, at, p.cols - at));
        }
    }
}

// One piece of grad_h.
template <int kType, bool kVec>
__device__ __forceinline__ void write_grad(const NormBackwardParams& p, int64_t row, int at, int valid, float r,
                                           float mean, const float (&g)[kPiece], const float (&n)[kPiece],
                                           const RawPiece<kType>& grad_h_in) {
    float out[kPiece], in[kPiece];
    unpack(grad_h_in, in);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) out[i] = r * (g[i] - n[i] * mean) + in[i];
    if (valid > 0) store_piece<kType, kVec>(row_at<kType>(p.grad_h, row, p.ld_grad_h), at, valid, out);
}

// One row's pieces of this lane, as loaded.
template <int kType, int kPieces>
struct NormRow {
    RawPiece<kType> g[kPieces], h[kPieces], in[kPieces];
    float r;
};

template <int kType, bool kVec, int kRowThreads, int kPieces>
__device__ __forceinline__ void fetch_row(const NormBackwardParams& p, int64_t row, int t, NormRow<kType, kPieces>& f) {
    f.r = p.rstd[row];
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
        const int at = (c * kRowThreads + t) * kPiece, valid = p.cols - at;
        f.g[c] = load_raw<kType, kVec>(row_at<kType>(p.grad_y, row, p.ld_grad_y), at, valid);
        f.h[c] = load_raw<kType, kVec>(row_at<kType>(p.h, row, p.ldh), at, valid);
        f.in[c] = p.grad_h_in ? load_raw<kType, kVec>(row_at<kType>(p.grad_h_in, row, p.ld_grad_h_in), at, valid)
                              : RawPiece<kType>{};
    }
}

// Rows blockIdx.x * R + (which of the workgroup's), and every gridDim.x * R on: the lanes keep the sums of grad_y n of
// their columns over all of them. The next row is on its way while a row's mean is taken.
template <int kType, bool kVec, int kRowWaves, int kPieces>
__global__ __launch_bounds__(threads_of(kRowWaves)) void norm_backward_kernel(const NormBackwardParams p) {
    constexpr int kRowThreads = 64 * kRowWaves;
    constexpr int kRows = threads_of(kRowWaves) / kRowThreads;
    __shared__ float lds[kRowWaves > 1 ? kRowWaves : kWaves * 64 * kPiece];
    const int t = threadIdx.x % kRowThreads;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kRowThreads;
    float dw[kPieces][kPiece] = {};
    RawPiece<kType> raw_w[kPieces];   // the weight's pieces where it has the activations' type
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
        const int at = (c * kRowThreads + t) * kPiece;
        raw_w[c] = weight_piece<kType, kVec>(p.weight, p.weight_fp32, at, p.cols - at);
    }
    NormRow<kType, kPieces> next;
    if (row < p.rows) fetch_row<kType, kVec, kRowThreads>(p, row, t, next);
    for (; row < p.rows; row += step) {
        NormRow<kType, kPieces> now = next;
        if (row + step < p.rows) fetch_row<kType, kVec, kRowThreads>(p, row + step, t, next);
        float g[kPieces][kPiece], n[kPieces][kPiece], sum = 0.0f;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            float w[kPiece];
            unpack(now.g[c], g[c]);
            unpack(now.h[c], n[c]);
            if (p.weight_fp32) load_piece<FEATHER_FP32, kVec>(p.weight, at, p.cols - at, w);
            else unpack(raw_w[c], w);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                n[c][i] *= now.r;
                dw[c][i] += g[c][i] * n[c][i];
                g[c][i] *= w[i];
                sum += g[c][i] * n[c][i];
            }
        }
        const float mean = row_sum<kRowWaves>(sum, lds) / static_cast<float>(p.cols);
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = (c * kRowThreads + t) * kPiece;
            write_grad<kType, kVec>(p, row, at, p.cols - at, now.r, mean, g[c], n[c], now.in[c]);
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
        store_piece<FEATHER_FP32, kVec>(part, at, p.cols - at, dw[c]);
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
            if (p.weight_fp32) load_piece<FEATHER_FP32, kVec>(p.weight, at, valid, w);
            else load_piece<kType, kVec>(p.weight, at, valid, w);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                n[i] *= r;
                g[i] *= w[i];
                sum += g[i] * n[i];
            }
            if (pass == 1) {
                write_grad<kType, kVec>(p, row, at, valid, r, mean, g, n,
                                        p.grad_h_in ? load_raw<kType, kVec>(
                                                          row_at<kType>(p.grad_h_in, row, p.ld_grad_h_in), at, valid)
                                                    : RawPiece<kType>{});
            }
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
    store_piece<FEATHER_FP32, kVec>(part, at, valid, dw);
}

// out[j] = the sum of part[., j]: a workgroup takes 16 columns (a 64-byte piece of each row), its 16 groups of 16 lanes every
// 16th row each with 8 rows in flight, joined in group order. 512 x 4096: 31 us with 64 columns and 4 groups a workgroup.
constexpr int kSumCols = 16;
constexpr int kSumGroups = kThreads / kSumCols;
constexpr int kSumAhead = 8;

template <int kType>
__global__ __launch_bounds__(kThreads) void sum_rows_kernel(const float* part, void* out, int64_t rows, int64_t cols,
                                                            int64_t ld) {
    __shared__ float lds[kSumGroups][kSumCols];
    const int group = threadIdx.x / kSumCols;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kSumCols + threadIdx.x % kSumCols;
    float s = 0.0f;
    if (col < cols) {
        for (int64_t i = group; i < rows; i += kSumGroups * kSumAhead) {
            float v[kSumAhead];
#pragma unroll
            for (int k = 0; k < kSumAhead; ++k) {
                const int64_t row = i + k * kSumGroups;
                v[k] = part[(row < rows ? row : rows - 1) * ld + col];   // no branch: 8 loads in flight
            }
#pragma unroll
            for (int k = 0; k < kSumAhead; ++k) s += i + k * kSumGroups < rows ? v[k] : 0.0f;
        }
    }
    lds[group][threadIdx.x % kSumCols] = s;
    __syncthreads();
    if (threadIdx.x >= kSumCols || col >= cols) return;
    s = lds[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < kSumGroups; ++k) s += lds[k][threadIdx.x];
    if constexpr (kType == FEATHER_FP32) static_cast<uint32_t*>(out)[col] = to_bits<kType>(s);
    else static_cast<uint16_t*>(out)[col] = static_cast<uint16_t>(to_bits<kType>(s));
}

constexpr int64_t kWaveCols = 2048;       // rows up to here are one wave's
constexpr int64_t kRegisterCols = 16384;  // and up to here in registers
constexpr int64_t kLongParts = 64;
constexpr int64_t kFewRows = 256;         // up to here (the CUs) a longer row has 16 waves

// Workgroups of the backward: 512 (two a CU), fewer where the rows are.
int64_t backward_groups(int64_t rows, int64_t cols) {
    if (cols > kRegisterCols) return rows < kLongParts ? rows : kLongParts;
    const int64_t groups = cols <= kWaveCols ? (rows + kWaves - 1) / kWaves : rows;
    return groups < 512 ? groups : 512;
}

// p from row `row` on.
NormParams from_row(NormParams p, int64_t row, int type) {
    const int bytes = type_bytes(type);
    p.x = static_cast<const uint8_t*>(p.x) + row * p.ldx * bytes;
    if (p.residual) p.residual = static_cast<const uint8_t*>(p.residual) + row * p.ld_residual * bytes;
    if (p.h) p.h = static_cast<uint8_t*>(p.h) + row * p.ldh * bytes;
    if (p.y) p.y = static_cast<uint8_t*>(p.y) + row * p.ldy * bytes;
    if (p.rstd) p.rstd += row;
    p.q = from_row(p.q, row);
    p.rows -= row;
    return p;
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

// Calls f<waves per row, pieces per lane>() for rows of `cols` values (at most kRegisterCols). Measured (us, 16-bit rows with a
// residual): as many waves as two pieces a lane make instead of four with three to eight, forward: 4112 x 5120 30.9 -> 30.0,
// 4096 x 8192 49.0 -> 47.0, 2048 x 12288 41.5 -> 34.9. The backward, which holds the next row too, has four waves up to 6144
// columns (4112 x 5120 37 against 43), then two pieces (4096 x 8192 81 -> 62, 2048 x 12288 71 -> 50), and four past 12288,
// where sixteen waves would leave a lane 128 registers (2048 x 16384 96).
template <bool kBackward, typename F>
void by_cols(int64_t rows, int64_t cols, F&& f) {
    using W1 = std::integral_constant<int, 1>;
    using W4 = std::integral_constant<int, kWaves>;
    using W8 = std::integral_constant<int, 8>;
    using W12 = std::integral_constant<int, 12>;
    using W16 = std::integral_constant<int, 16>;
    using P1 = std::integral_constant<int, 1>;
    using P2 = std::integral_constant<int, 2>;
    using P3 = std::integral_constant<int, 3>;
    using P4 = std::integral_constant<int, 4>;
    if (cols <= 512) f(W1{}, P1{});
    else if (cols <= 1024) f(W1{}, P2{});
    else if (cols <= 2048) f(W1{}, P4{});
    else if (rows <= kFewRows && cols <= 8192) f(W16{}, P1{});
    else if (cols <= 4096) f(W4{}, P2{});
    else if constexpr (kBackward) {
        if (cols <= 6144) f(W4{}, P3{});
        else if (cols <= 8192) f(W8{}, P2{});
        else if (cols <= 12288) f(W12{}, P2{});
        else f(W8{}, P4{});
    } else {
        if (rows <= kFewRows) f(W16{}, P2{});
        else if (cols <= 5120) f(std::integral_constant<int, 5>{}, P2{});
        else if (cols <= 6144) f(std::integral_constant<int, 6>{}, P2{});
        else if (cols <= 8192) f(W8{}, P2{});
        else if (cols <= 10240) f(std::integral_constant<int, 10>{}, P2{});
        else if (cols <= 12288) f(W12{}, P2{});
        else f(W16{}, P2{});
    }
}

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
    const bool vec = cols % kPiece == 0 && rows_on_16(x, ldx, type) && on_16(weight) &&
                     (!residual || (rows_on_16(residual, ld_residual, type) && rows_on_16(h, ldh, type))) &&
                     (y ? rows_on_16(y, ldy, type) : (on_16(codes) && ld_codes % 8 == 0));
    const auto launch = [&](auto kernel, int threads, int64_t group_rows) {
        const int64_t most = kMaxThreads / threads * group_rows;   // rows of a launch
        for (int64_t row = 0; row < rows; row += most) {
            NormParams part = from_row(p, row, type);
            part.rows = std::min(part.rows, most);
            kernel<<<static_cast<uint32_t>((part.rows + group_rows - 1) / group_rows), threads, 0, stream>>>(part);
        }
    };
    by_type(type, vec, [&](auto t, auto v) {
        if (cols > kRegisterCols) {
            launch(norm_kernel<t(), v(), kWaves, 0>, kThreads, 1);
            return;
        }
        by_cols<false>(rows, cols, [&](auto waves, auto pieces) {
            launch(norm_kernel<t(), v(), waves(), pieces()>, threads_of(waves()), waves() == 1 ? kWaves : 1);
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
    if (cols > kRegisterCols && rows > kMaxThreads / kThreads) return false;
    const NormBackwardParams p{grad_y, grad_h_in, h, weight, rstd, grad_h, part, ld_grad_y, ld_grad_h_in, ldh,
                               ld_grad_h, rows, static_cast<int32_t>(cols), weight_fp32};
    const bool vec = cols % kPiece == 0 && on_16(part) && rows_on_16(grad_y, ld_grad_y, type) && rows_on_16(h, ldh, type) &&
                     rows_on_16(grad_h, ld_grad_h, type) && on_16(weight) &&
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
        by_cols<true>(rows, cols, [&](auto waves, auto pieces) {
            norm_backward_kernel<t(), v(), waves(), pieces()><<<groups, threads_of(waves()), 0, stream>>>(p);
        });
    });
    return true;
}

extern "C" bool feather_sum_rows(const float* part, void* out, int type, int64_t rows, int64_t cols,
                                 hipStream_t stream) {
    if (!part || !out || !type_ok(type) || rows < 1 || cols < 1 || !aligned_to_type(out, type)) return false;
    constexpr int64_t kMost = kMaxThreads / kThreads * kSumCols;   // columns of a launch
    by_type(type, true, [&](auto t, auto) {
        for (int64_t col = 0; col < cols; col += kMost) {
            const int64_t here = std::min(cols - col, kMost);
            const auto groups = static_cast<uint32_t>((here + kSumCols - 1) / kSumCols);
            sum_rows_kernel<t()><<<groups, kThreads, 0, stream>>>(
                part + col, static_cast<uint8_t*>(out) + col * type_bytes(type), rows, here, cols);
        }
    });
    return true;
}
