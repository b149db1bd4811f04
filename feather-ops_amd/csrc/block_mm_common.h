// What the kernels of the block-scaled fp8 product share (include/feather_block_ops.h):
//   c[m, n] = round( sum over blocks k of sa[m, k] sb[n, k] * (sum over the block of a[m, .] b[n, .]) + bias[n] )
//
// A block of 128 is the contraction of one v_mfma_f32_16x16x128_f8f6f4, so each MFMA starts from zero and its 16 x 16
// result is added to the fp32 accumulators times the block's scales: one multiply-add per output and block, on the vector
// unit while the matrix unit runs the next block.
//
// Fragment layout (wave64). The MFMA's first operand carries 16 rows of b and its second 16 rows of a, so lane l ends up
// with output row l % 16 and the 4 consecutive output columns 4 (l / 16) + {0..3} of a 16 x 16 tile: one value of sa per
// lane, and one 8- or 16-byte store. Lane group g = l / 16 feeds bytes 16 g .. + 15 and 64 + 16 g .. + 15 of the block for
// both operands; any assignment that both share gives the same sum, and this one reads whole half lines of memory.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "block_common.h"
#include "scaled_mm_kernels.h"
#include "split_join.h"

namespace feather {

using i32x8 = int32_t __attribute__((ext_vector_type(8)));

struct BlockMmParams {
    const uint8_t* a;
    const uint8_t* b;
    const float* a_scale;
    const float* b_scale;
    int64_t lda, ldb, as_row, as_block, bs_row, bs_block;
    int32_t M, N, K;
    int32_t splits;
    const void* bias;
    void* c;
    int64_t ldc;
    int32_t out_type;
    uint32_t* split_ctr;
    uint8_t* split_part;
};

// A 16 x 16 x 128 product from zero. Formats: 0 e4m3fn, 1 e5m2.
template <bool kAE5M2, bool kBE5M2>
__device__ __forceinline__ f32x4 mfma_block(i32x8 b, i32x8 a) {
    const f32x4 zero{0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, zero, kBE5M2, kAE5M2, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8 join16(u32x4 lo, u32x4 hi) {
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The first `valid` of 16 bytes, the rest zero.
__device__ __forceinline__ u32x4 keep_bytes(u32x4 v, int valid) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int n = valid - 4 * d;
        const uint32_t mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        v[d] &= mask;
    }
    return v;
}

// Rows row0 .. of a matrix as a buffer that ends with the last of at most `rows` of them (up to the last whole dword): what
// lies past it reads as zero.
__device__ __forceinline__ rsrc_t rows_rsrc(const uint8_t* base, int64_t ld, int row0, int total, int rows, int K) {
    const int here = total - row0 < rows ? total - row0 : rows;
    const uint32_t bytes = here > 0 ? static_cast<uint32_t>(here - 1) * static_cast<uint32_t>(ld) + ((K + 3) & ~3) : 0u;
    return make_rsrc(base + row0 * ld, bytes);
}

// Four outputs of row m at columns n .. n + 3: bias added in fp32, rounded once.
__device__ __forceinline__ void store_out(const BlockMmParams& p, int m, int n, f32x4 v) {
    if (m >= p.M || n >= p.N) return;
    const int valid = p.N - n;
    const int64_t at = static_cast<int64_t>(m) * p.ldc + n;
    const auto go = [&](auto type) {
        constexpr int kType = type();
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < valid) {
                    if constexpr (kType == FEATHER_FP32) v[i] += static_cast<const float*>(p.bias)[n + i];
                    else v[i] += to_float<kType>(static_cast<const uint16_t*>(p.bias)[n + i]);
                }
        }
        if constexpr (kType == FEATHER_FP32) {
            auto* out = static_cast<float*>(p.c) + at;
            if (valid >= 4) {
                store_any(out, v);
            } else {
                for (int i = 0; i < 3; ++i)
                    if (i < valid) out[i] = v[i];
            }
        } else {
            auto* out = static_cast<uint16_t*>(p.c) + at;
            if (valid >= 4) {
                store_any(out, u32x2{pack2<kType>(v[0], v[1]), pack2<kType>(v[2], v[3])});
            } else {
                for (int i = 0; i < 3; ++i)
                    if (i < valid) out[i] = static_cast<uint16_t>(to_bits<kType>(v[i]));
            }
        }
    };
    if (p.out_type == FEATHER_BF16) go(std::integral_constant<int, FEATHER_BF16>{});
    else if (p.out_type == FEATHER_FP16) go(std::integral_constant<int, FEATHER_FP16>{});
    else go(std::integral_constant<int, FEATHER_FP32>{});
}

// acc += t * sa * sb for four columns; sb the same for all of them or one each.
__device__ __forceinline__ void add_scaled(f32x4& acc, const f32x4 t, float s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(t[i], s, acc[i]);
}

__device__ __forceinline__ void add_scaled(f32x4& acc, const f32x4 t, const f32x4 s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(t[i], s[i], acc[i]);
}

}  // namespace feather
