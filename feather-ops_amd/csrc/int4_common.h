// 4-bit weights with group scales (include/feather_linear_ops.h): w[n, k] = (q[n, k] - z[n, k / group]) s[n, k / group], codes q of
// 0 .. 15 two to a byte, the even k in the low half.
//
// A dword holds 8 codes of consecutive k. They become 16-bit values two at a time, in the order 0 4 1 5 2 6 3 7, by putting a
// code's bits into the mantissa of a power of two: fp16 1024 + q, whose 1024 + z is taken off again, exactly; bf16 128 + q, which
// stays (there is no packed bf16 arithmetic): its 128 + z, times the sum of x, is taken off the group's sum in fp32.
// Activations are put into the same order.
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

// What decode8 keeps in registers: the powers of two that codes are put into and, fp16, what is taken off again: of the low
// nibbles 1024 + z, of the high ones, which stay in their place, 64 + z.
template <bool kBf16>
struct Decode {
    uint32_t one, low, high;

    __device__ __forceinline__ void init() {
        one = kBf16 ? 0x43004300u : 0x64006400u;   // 128, 1024
        asm volatile("" : "+v"(one));              // (the compiler would rather spend two instructions on literals)
        low = 0x64086408u;                         // 1032
        high = 0x54805480u;                        // 72
    }
    // fp16: codes of a row with zero point z.
    __device__ __forceinline__ void set_zero(uint32_t z) {
        z |= z << 16;
        low = 0x64006400u | z;
        high = 0x54005400u | z << 4;
    }
    // 8 codes -> 8 values code - z (fp16) or code + 128 (bf16), in the order 0 4 1 5 2 6 3 7.
    __device__ __forceinline__ half8 operator()(uint32_t w) const {
        constexpr uint32_t kLow = 0x000f000fu;
        const auto insert = [&](uint32_t v, uint32_t mask) { return (v & mask) | one; };
        if constexpr (kBf16) {
            return __builtin_bit_cast(half8, u32x4{insert(w, kLow), insert(w >> 4, kLow), insert(w >> 8, kLow), insert(w >> 12, kLow)});
        } else {
            const uint32_t u = w >> 8;
            const half2v part{static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
            const auto at_low = [&](uint32_t v) {
                return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, insert(v, kLow)) - __builtin_bit_cast(half2v, low));
            };
            const auto at_high = [&](uint32_t v) {   // 1024 + 16 q
                return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, insert(v, kLow << 4)), part,
                                                                              -__builtin_bit_cast(half2v, high)));
            };
            return __builtin_bit_cast(half8, u32x4{at_low(w), at_high(w), at_low(u), at_high(u)});
        }
    }
};

// 8 activations into the codes' order.
__device__ __forceinline__ half8 order8(u32x4 v) {
    constexpr uint32_t kLow = perm_sel(0, 1, 4, 5), kHigh = perm_sel(2, 3, 6, 7);   // of (v_perm's second, first) operand
    return __builtin_bit_cast(half8, u32x4{__builtin_amdgcn_perm(v[2], v[0], kLow), __builtin_amdgcn_perm(v[2], v[0], kHigh),
                                           __builtin_amdgcn_perm(v[3], v[1], kLow), __builtin_amdgcn_perm(v[3], v[1], kHigh)});
}

// bf16: 8 times -136, what takes a code + 128 to code - 8, or 1.
template <bool kOffset>
__device__ __forceinline__ half8 constant8() {
    constexpr uint32_t k = kOffset ? 0xc308c308u : 0x3f803f80u;
    return __builtin_bit_cast(half8, u32x4{k, k, k, k});
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

// Where a lane reads its 4 columns' scales and zero points in a group's row (which has 4 values at least), and by how many values
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

__device__ __forceinline__ f32x4 zeros4(uint32_t raw, uint32_t shift) {
    raw >>= 8 * shift & 31;
    return f32x4{static_cast<float>(raw & 255u), static_cast<float>(raw >> 8 & 255u), static_cast<float>(raw >> 16 & 255u),
                 static_cast<float>(raw >> 24)};
}

}  // namespace feather
