// 4-bit weights with group scales (include/feather_linear_ops.h): w[n, k] = (q[n, k] - z[n, k / group]) s[n, k / group], codes q of
// 0 .. 15 two to a byte, the even k in the low half.
//
// A dword holds 8 codes of consecutive k. They become 16-bit values q - z two at a time, exactly: fp16 by putting a code's bits into
// the mantissa of a power of two, 1024 + q, whose 1024 + z is taken off again; bf16, which has no packed arithmetic, by way of a conversion
// from 8 bits. Activations are put into the order that they come in.
#pragma once

#include "linear_common.h"

namespace feather {

struct Int4Params : LinearParams {   // b: unused
    const uint8_t* codes;       // [N, ceil(K / 2)] bytes, rows ld_codes apart
    const uint16_t* scale;      // [groups, N] of a's type: group by group, ld_scale apart
    const uint8_t* zero;        // [groups, N], ld_zero apart; or null: 8
    int64_t ld_codes, ld_scale, ld_zero;
    int32_t group;              // 32, 64 or 128
};

// What decoding keeps in registers. fp16: the power of two that codes are put into and what is taken off again: of the low nibbles
// 1024 + z, of the high ones, which stay in their place, 64 + z. bf16: the zero point.
//
// Values go to the matrix units exactly, so that sums have fp32's accuracy and x may be anything, infinities too. For 8 codes fp16 takes
// 9 instructions and bf16 13, with zero points 19. (codes + 128, whose 128 + z times the sum of x comes off again, take bf16 7, lose 5 bits
// of a sum and fail on infinities: one row of 4096 -> 14336 gated 15.2 us, now 16.8, 24 rows 20.6 both, 64 rows 45.0 and 45.4. Other
// exact ways: by fp16 and two conversions 19.7, by fp32 18.0.)
template <bool kBf16>
struct Decode {
    // bf16: a value is (q - z) / kUnit, so that no sum of a group, 128 values of up to 15 times x, passes fp32's range. Outputs are
    // multiplied by it.
    static constexpr float kUnit = kBf16 ? 2048.0f : 1.0f;
    uint32_t one, low, high;
    float zero;

    __device__ __forceinline__ void init() {
        one = 0x64006400u;              // 1024
        asm volatile("" : "+v"(one));   // (the compiler would rather spend two instructions on literals)
        low = 0x64086408u;              // 1032
        high = 0x54805480u;             // 72
        zero = 8.0f / kUnit;
    }
    // Codes of a row with zero point z.
    __device__ __forceinline__ void set_zero(uint32_t z) {
        if constexpr (kBf16) {
            zero = static_cast<float>(z) / kUnit;
        } else {
            z |= z << 16;
            low = 0x64006400u | z;
            high = 0x54005400u | z << 4;
        }
    }
    // 8 codes -> 8 values code - z, in order8's order.
    template <bool kZeros>
    __device__ __forceinline__ half8 values(uint32_t w) const {
        if constexpr (kBf16 && kZeros) {
            const uint32_t codes[2] = {w & 0x0f0f0f0fu, w >> 4 & 0x0f0f0f0fu};   // even, odd
            u32x4 out;
#pragma unroll
            for (int i = 0; i < 2; ++i) {   // a byte, read as e4m3, is q / 512
                const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[i], 512.0f / kUnit, false);
                const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[i], 512.0f / kUnit, true);
                out[2 * i] = pack2<FEATHER_BF16>(a[0] - zero, a[1] - zero);
                out[2 * i + 1] = pack2<FEATHER_BF16>(b[0] - zero, b[1] - zero);
            }
            return __builtin_bit_cast(half8, out);
        } else if constexpr (kBf16) {
            // q - 8 as sign and magnitude, which together, in a byte's ends, are e4m3: below 8 the magnitude is 8 - q, the other bits' complement + 1
            const uint32_t sign = ~w & 0x88888888u;
            const uint32_t below = sign >> 3;
            const uint32_t size = ((w & 0x77777777u) ^ (sign - below)) + below;
            const uint32_t even = (size & 0x0f0f0f0fu) | (sign << 4 & 0xf0f0f0f0u);
            const uint32_t odd = (size >> 4 & 0x0f0f0f0fu) | (sign & 0xf0f0f0f0u);
            const auto two = [&](uint32_t codes, auto high) {
                return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 512.0f / kUnit, high()));
            };
            return __builtin_bit_cast(half8, u32x4{two(even, std::false_type{}), two(even, std::true_type{}), two(odd, std::false_type{}),
                                                   two(odd, std::true_type{})});
        } else {
            constexpr uint32_t kLow = 0x000f000fu;
            const auto insert = [&](uint32_t v, uint32_t mask) { return __builtin_bit_cast(half2v, (v & mask) | one); };
            const uint32_t u = w >> 8;
            const half2v part{static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
            const auto at_low = [&](uint32_t v) {
                return __builtin_bit_cast(uint32_t, insert(v, kLow) - __builtin_bit_cast(half2v, low));
            };
            const auto at_high = [&](uint32_t v) {   // 1024 + 16 q
                return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(insert(v, kLow << 4), part, -__builtin_bit_cast(half2v, high)));
            };
            return __builtin_bit_cast(half8, u32x4{at_low(w), at_high(w), at_low(u), at_high(u)});
        }
    }
};

// 8 activations into the codes' order: fp16 0 4 1 5 2 6 3 7, bf16 0 2 4 6 1 3 5 7.
template <bool kBf16>
__device__ __forceinline__ half8 order8(u32x4 v) {
    constexpr uint32_t kLow = perm_sel(0, 1, 4, 5), kHigh = perm_sel(2, 3, 6, 7);   // of (v_perm's second, first) operand
    if constexpr (kBf16) {
        return __builtin_bit_cast(half8, u32x4{__builtin_amdgcn_perm(v[1], v[0], kLow), __builtin_amdgcn_perm(v[3], v[2], kLow),
                                               __builtin_amdgcn_perm(v[1], v[0], kHigh), __builtin_amdgcn_perm(v[3], v[2], kHigh)});
    }
    return __builtin_bit_cast(half8, u32x4{__builtin_amdgcn_perm(v[2], v[0], kLow), __builtin_amdgcn_perm(v[2], v[0], kHigh),
                                           __builtin_amdgcn_perm(v[3], v[1], kLow), __builtin_amdgcn_perm(v[3], v[1], kHigh)});
}

// Dword d of lane row r to dword r of lane row d: a lane that loaded 32 consecutive k's of its row then holds, as dword s, the
// k = 32 s + 8 g .. + 7 that MFMA s wants of lane row g.
__device__ __forceinline__ u32x4 transpose_rows(u32x4 v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{c[0], c[1], d[0], d[1]};
}

// Where a lane reads its 4 columns' scales in a group's row (which has 4 values at least), and by how many values
// the last columns' are shifted: nothing past the row is read.
struct ScaleAt {
    uint32_t from, shift;
};

__device__ __forceinline__ ScaleAt scale_at(int n, int N) {
    const int last = N > 4 ? N - 4 : 0;
    const int from = n < last ? n : last;
    return {static_cast<uint32_t>(from), static_cast<uint32_t>(n - from)};
}

template <bool kBf16>
__device__ __forceinline__ f32x4 scales4(u32x2 raw, uint32_t shift) {
    const uint64_t v = (static_cast<uint64_t>(raw[1]) << 32 | raw[0]) >> (16 * shift & 63);
    const auto lo = static_cast<uint32_t>(v), hi = static_cast<uint32_t>(v >> 32);
    constexpr int kType = kTypeOf<kBf16>;
    if constexpr (kBf16) {
        return f32x4{to_float<kType>(lo & 0xffffu), __builtin_bit_cast(float, lo & 0xffff0000u), to_float<kType>(hi & 0xffffu),
                     __builtin_bit_cast(float, hi & 0xffff0000u)};
    }
    return f32x4{to_float<kType>(lo & 0xffffu), to_float<kType>(lo >> 16), to_float<kType>(hi & 0xffffu), to_float<kType>(hi >> 16)};
}

}  // namespace feather
