// What the 16-bit and 4-bit products share (include/feather_linear_ops.h): operands, the gated epilogue's arithmetic and the
// ways outputs leave.
//
// Fragment layout (v_mfma_f32_16x16x32, wave64): the first operand carries 16 rows of b (output columns), the second 16 rows of
// a, so lane l ends up with output row l % 16 and the 4 consecutive columns 4 (l / 16) + {0..3}. Lane group g = l / 16 feeds k =
// 8 g .. + 7 of 32 for both.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "activation.h"
#include "block_common.h"
#include "scaled_mm_kernels.h"
#include "split_join.h"

namespace feather {

enum class Form { kPlain, kGated, kGatedKeep };   // what becomes of the sums: outputs; gate * up; and both kept in fp32

struct LinearParams {
    const uint16_t* a;      // [M, K], or [K, M] where transposed
    const uint16_t* b;      // [N, K] ([2 N, K] gated: the gates' rows, then the ups'), or [K, N] where transposed
    int64_t lda, ldb;       // elements
    int32_t M, N, K;
    int32_t m_first, n_first;   // tiles: the outputs where this launch starts, and how many tiles there are
    int32_t tiles_m, tiles_n;
    int32_t splits;
    const void* bias;       // N values ([2 N] gated) of the operands' type, or null
    void* c;                // [M, N]
    int64_t ldc;
    float* h;               // kGatedKeep: [M, 2 N], the sums with their bias
    int64_t ldh;
    uint32_t* split_ctr;
    uint8_t* split_part;
    int32_t act;
};

template <bool kBf16>
constexpr int kTypeOf = kBf16 ? FEATHER_BF16 : FEATHER_FP16;

// Bias values n .. n + 3 of `total`, zero where there are none.
template <bool kBf16>
__device__ __forceinline__ f32x4 bias4(const void* bias, int64_t n, int64_t total) {
    f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
    if (!bias) return v;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < total) v[e] = to_float<kTypeOf<kBf16>>(static_cast<const uint16_t*>(bias)[n + e]);
    return v;
}

template <int kAct>
__device__ __forceinline__ f32x4 gate4(f32x4 gate, f32x4 up) {
#pragma unroll
    for (int e = 0; e < 4; ++e) up[e] *= activate<kAct>(gate[e]);
    return up;
}

// A wave's outputs, rounded, as rows in LDS of its own: they leave as pieces of 16 bytes, neighbouring lanes side by side, at any
// alignment. (Straight from the fragments each store would need its own code for the matrix's edges.)
template <int RM, int kFragments>
struct OutStage {
    static constexpr int kRowBytes = 32 * kFragments;
    static constexpr int kPitch = kRowBytes + 16;   // the rows' writes of a column fall on different banks
    static constexpr int kBytes = 16 * RM * kPitch;
};

template <int RM, int kFragments>
__device__ __forceinline__ void store_staged(const LinearParams& p, int row0, int col0, int lane, const uint8_t* own) {
    using O = OutStage<RM, kFragments>;
    constexpr int kLanes = O::kRowBytes / 16;   // of a row
    __builtin_amdgcn_s_waitcnt(kLgkm0Imm);      // the wave reads what it wrote itself
    const int n = col0 + lane % kLanes * 8;
    const int valid = p.N - n;
    if (valid <= 0) return;
#pragma unroll 4
    for (int r = lane / kLanes; r < 16 * RM; r += 64 / kLanes) {
        const int m = row0 + r;
        if (m >= p.M) break;
        const u32x4 v = *reinterpret_cast<const u32x4*>(own + r * O::kPitch + lane % kLanes * 16);
        uint16_t* const out = static_cast<uint16_t*>(p.c) + static_cast<int64_t>(m) * p.ldc + n;
        if (valid >= 8) {
            store_any(out, v);
        } else {
#pragma unroll 1
            for (int e = 0; e < valid; ++e) {
                const uint32_t word = e < 4 ? (e < 2 ? v[0] : v[1]) : (e < 6 ? v[2] : v[3]);
                out[e] = static_cast<uint16_t>(word >> (16 * (e % 2)));
            }
        }
    }
}

// A wave's RM x RN sums to outputs. Plain: fragment j is columns col0 + 16 j ..; gated: fragments 2 q and 2 q + 1 are the gate
// and up of columns col0 + 16 q ...
template <Form kForm, bool kBf16, int RM, int RN, int kAct>
__device__ __forceinline__ void finish_as(const LinearParams& p, f32x4 (&acc)[RM][RN], int row0, int col0, int lane,
                                          uint8_t* own) {
    constexpr bool kGated = kForm != Form::kPlain;
    constexpr int kFragments = kGated ? RN / 2 : RN;
    using O = OutStage<RM, kFragments>;
    const int c4 = 4 * (lane / 16);
    const int r16 = lane % 16;
    [[maybe_unused]] rsrc_t h_rsrc;
    if constexpr (kForm == Form::kGatedKeep) {
        const int rows = p.M - row0 < 16 * RM ? p.M - row0 : 16 * RM;
        h_rsrc = make_rsrc(p.h + row0 * p.ldh, rows > 0 ? static_cast<uint32_t>(rows) * static_cast<uint32_t>(p.ldh * 4) : 0u);
    }
#pragma unroll
    for (int q = 0; q < kFragments; ++q) {
        const int n = col0 + 16 * q + c4;
        const f32x4 bias = bias4<kBf16>(p.bias, n, p.N);
        [[maybe_unused]] f32x4 bias_up;
        if constexpr (kGated) bias_up = bias4<kBf16>(p.bias, p.N + n, n < p.N ? 2 * p.N : 0);
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            f32x4 v;
            if constexpr (kGated) {
                const f32x4 gate = acc[i][2 * q] + bias;
                const f32x4 up = acc[i][2 * q + 1] + bias_up;
                if constexpr (kForm == Form::kGatedKeep) {
                    // rows of h hold both halves padded to 8 columns
                    const int half = (p.N + 7) & ~7;
                    const uint32_t at = static_cast<uint32_t>(16 * i + r16) * static_cast<uint32_t>(p.ldh * 4) + static_cast<uint32_t>(n) * 4u;
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, gate), h_rsrc,
                                                           static_cast<int>(n < half ? at : kOob), 0, 0);
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, up), h_rsrc,
                                                           static_cast<int>(n < half ? at : kOob), half * 4, 0);
                }
                v = gate4<kAct>(gate, up);
            } else {
                v = acc[i][q] + bias;
            }
            *reinterpret_cast<u32x2*>(own + (16 * i + r16) * O::kPitch + 32 * q + 2 * c4) =
                u32x2{pack2<kTypeOf<kBf16>>(v[0], v[1]), pack2<kTypeOf<kBf16>>(v[2], v[3])};
        }
    }
    store_staged<RM, kFragments>(p, row0, col0, lane, own);
}

template <Form kForm, bool kBf16, int RM, int RN>
__device__ __forceinline__ void finish(const LinearParams& p, f32x4 (&acc)[RM][RN], int row0, int col0, int lane, uint8_t* own) {
    if constexpr (kForm == Form::kPlain) {
        finish_as<kForm, kBf16, RM, RN, kSilu>(p, acc, row0, col0, lane, own);
    } else {
        if (p.act == kSilu) finish_as<kForm, kBf16, RM, RN, kSilu>(p, acc, row0, col0, lane, own);
        else if (p.act == kGelu) finish_as<kForm, kBf16, RM, RN, kGelu>(p, acc, row0, col0, lane, own);
        else finish_as<kForm, kBf16, RM, RN, kGeluTanh>(p, acc, row0, col0, lane, own);
    }
}

}  // namespace feather
