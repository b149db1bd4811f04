// What the operators with one scale for each block of 128 values share (include/feather_block_ops.h): 8-value pieces of
// rows, and the quantization of blocks.
//
// A row is handled in pieces of 8 consecutive values, one per lane and step, so a block of 128 is the 16 lanes of one DPP
// row: its largest value takes four row rotations and no LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "feather_block_ops.h"

namespace feather {

constexpr int kBlock = 128;           // values per scale
constexpr int kPiece = 8;             // values per lane and step
constexpr uint32_t kLeastBits = 27u << 23;  // 2^-100: the least a block's largest value counts as

using u32x4v = uint32_t __attribute__((ext_vector_type(4)));
using u32x2v = uint32_t __attribute__((ext_vector_type(2)));

// Bytes of one value of `type`.
__host__ __device__ constexpr int type_bytes(int type) { return type == FEATHER_FP32 ? 4 : 2; }

template <int kType>
__device__ __forceinline__ float to_float(uint32_t bits) {
    if constexpr (kType == FEATHER_BF16) return __builtin_bit_cast(float, bits << 16);
    if constexpr (kType == FEATHER_FP16)
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
    return __builtin_bit_cast(float, bits);
}

// v rounded to the type (nearest even; subnormals and NaN kept), as its bits.
template <int kType>
__device__ __forceinline__ uint32_t to_bits(float v) {
    if constexpr (kType == FEATHER_BF16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
    if constexpr (kType == FEATHER_FP16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
    return __builtin_bit_cast(uint32_t, v);
}

// Two values rounded to a 16-bit type and packed, the first one lowest.
template <int kType>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    using f32x2 = float __attribute__((ext_vector_type(2)));
    if constexpr (kType == FEATHER_BF16) {
        using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
    } else {
        using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), f16x2));
    }
}

// A piece's bits as they are in memory: a value that is loaded well before it is used holds half the registers of its 8
// floats, and its conversion does not wait for it early.
template <int kType>
struct RawPiece {
    static constexpr int kWords = kType == FEATHER_FP32 ? 8 : 4;
    uint32_t w[kWords];
};

// 16 or 8 bytes from or to an address of any alignment, one access (the GPU runs in its unaligned mode, as HSA sets it).
template <typename V>
__device__ __forceinline__ V load_any(const void* p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}

template <typename V>
__device__ __forceinline__ void store_any(void* p, V v) {
    __builtin_memcpy(p, &v, sizeof(V));
}

// The piece without its first `n` (0 .. 8) values, the rest moved down and zeros behind.
template <int kType>
__device__ __forceinline__ RawPiece<kType> drop_values(RawPiece<kType> raw, int n) {
    constexpr int kWords = RawPiece<kType>::kWords;
    const int words = kType == FEATHER_FP32 ? n : n / 2;
#pragma unroll
    for (int by = kWords; by >= 1; by /= 2) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw.w[i] = words & by ? (i + by < kWords ? raw.w[i + by] : 0u) : raw.w[i];
    }
    if (kType != FEATHER_FP32 && n % 2) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw.w[i] = raw.w[i] >> 16 | (i + 1 < kWords ? raw.w[i + 1] << 16 : 0u);
    }
    return raw;
}

// The 8 values at element `at` of the row `row`, of which `valid` (may be <= 0 or > 8) are there; the others are zero. The row
// has at + valid values, no fewer: what lies past them is not read. No load
// is a branch, so that all of a lane's loads are in flight together. (Behind branches each waited for the one before: the
// norm of one row of 14336, 7 pieces a lane, took 10.7 us.)
// kVec: whole pieces are 16-byte aligned and rows are whole pieces (valid <= 0 or >= 8): a lane past the end reads the
// row's first piece and drops it. Otherwise pieces of any alignment; one past or over the row's end reads the row's last 8
// values and drops those before it; rows shorter than a piece go value by value. (Value by value throughout, the norm of
// 4096 x 4097 took 76 us, with 4096 columns 25.)
template <int kType, bool kVec>
__device__ __forceinline__ RawPiece<kType> load_raw(const void* row, int at, int valid) {
    constexpr int kWords = RawPiece<kType>::kWords;
    RawPiece<kType> raw;
    if (kVec || at + valid >= kPiece) {
        const int over = kVec ? 0 : min(kPiece, max(0, kPiece - valid));   // values of the piece past the row's end
        const int from = kVec ? (valid > 0 ? at : 0) : min(at, at + valid - kPiece);
        const uint8_t* p = static_cast<const uint8_t*>(row) + static_cast<int64_t>(from) * type_bytes(kType);
#pragma unroll
        for (int h = 0; h < kWords / 4; ++h) {
            const u32x4v v = kVec ? reinterpret_cast<const u32x4v*>(p)[h] : load_any<u32x4v>(p + 16 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) raw.w[4 * h + i] = !kVec || valid > 0 ? v[i] : 0u;
        }
        return kVec || over == 0 ? raw : drop_values(raw, over);
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw.w[i] = 0;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
        if (i < valid) {
            if constexpr (kType == FEATHER_FP32) raw.w[i] = static_cast<const uint32_t*>(row)[at + i];
            else raw.w[i / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(row)[at + i]) << (16 * (i % 2));
        }
    }
    return raw;
}

template <int kType>
__device__ __forceinline__ void unpack(const RawPiece<kType>& raw, float (&v)[kPiece]) {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
        if constexpr (kType == FEATHER_FP32) v[i] = __builtin_bit_cast(float, raw.w[i]);
        else if constexpr (kType == FEATHER_BF16)
            v[i] = __builtin_bit_cast(float, i % 2 ? raw.w[i / 2] & 0xffff0000u : raw.w[i / 2] << 16);
        else v[i] = to_float<kType>(i % 2 ? raw.w[i / 2] >> 16 : raw.w[i / 2] & 0xffffu);
    }
}

template <int kType, bool kVec>
__device__ __forceinline__ void load_piece(const void* row, int at, int valid, float (&v)[kPiece]) {
    unpack(load_raw<kType, kVec>(row, at, valid), v);
}

template <int kType, bool kVec>
__device__ __forceinline__ void store_piece(void* row, int at, int valid, const float (&v)[kPiece]) {
    uint8_t* out = static_cast<uint8_t*>(row) + static_cast<int64_t>(at) * type_bytes(kType);
    if (valid >= kPiece) {
        u32x4v words[type_bytes(kType) / 2];
        if constexpr (kType == FEATHER_FP32) {
            words[0] = u32x4v{to_bits<kType>(v[0]), to_bits<kType>(v[1]), to_bits<kType>(v[2]), to_bits<kType>(v[3])};
            words[1] = u32x4v{to_bits<kType>(v[4]), to_bits<kType>(v[5]), to_bits<kType>(v[6]), to_bits<kType>(v[7])};
        } else {
            words[0] = u32x4v{pack2<kType>(v[0], v[1]), pack2<kType>(v[2], v[3]), pack2<kType>(v[4], v[5]),
                              pack2<kType>(v[6], v[7])};
        }
#pragma unroll
        for (int h = 0; h < type_bytes(kType) / 2; ++h) {
            if constexpr (kVec) reinterpret_cast<u32x4v*>(out)[h] = words[h];
            else store_any(out + 16 * h, words[h]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
        if (i < valid) {
            if constexpr (kType == FEATHER_FP32) reinterpret_cast<uint32_t*>(out)[i] = to_bits<kType>(v[i]);
            else reinterpret_cast<uint16_t*>(out)[i] = static_cast<uint16_t>(to_bits<kType>(v[i]));
        }
    }
}

// ---- reductions without LDS -------------------------------------------------------------------------------

template <int kRotate>
__device__ __forceinline__ uint32_t row_ror(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x120 + kRotate, 0xf, 0xf, true));
}

// The largest of 16 lanes' values, in each of them.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, row_ror<8>(v));
    v = max(v, row_ror<4>(v));
    v = max(v, row_ror<2>(v));
    return max(v, row_ror<1>(v));
}

__device__ __forceinline__ float add_ror(float v, uint32_t r) { return v + __builtin_bit_cast(float, r); }

// The wave's sum, in every lane.
__device__ __forceinline__ float sum64(float v) {
    v = add_ror(v, row_ror<8>(__builtin_bit_cast(uint32_t, v)));
    v = add_ror(v, row_ror<4>(__builtin_bit_cast(uint32_t, v)));
    v = add_ror(v, row_ror<2>(__builtin_bit_cast(uint32_t, v)));
    v = add_ror(v, row_ror<1>(__builtin_bit_cast(uint32_t, v)));
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// ---- quantization -------------------------------------------------------------------------------------------

// |v| as bits: ordered like the values, infinity above them and NaN above infinity, so an unsigned maximum keeps NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t max_bits(const float (&v)[kPiece]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) m = max(m, abs_bits(v[i]));
    return m;
}

constexpr float kLeast = 0x1p-100f;

// What takes a block's values to codes: a product with L / amax in place of the quotient by amax / L, one division a block
// instead of one a value. The product of the largest value is at most L (1 + 2^-22), which rounds to L, so codes need no
// clamp. One term for values that were computed in fp32 and are off by as much themselves.
struct Factor {
    float hi;
    // Of a block whose largest magnitude is amax; the scale. (As bits NaN is above every number.)
    __device__ __forceinline__ float set(float amax, float largest, float, float) {
        amax = __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, amax), kLeastBits));
        hi = largest / amax;
        return amax / largest;
    }
    __device__ __forceinline__ float operator()(float v) const { return v * hi; }
};

// L / amax as hi + lo, within 2^-46 of it, for values that are given: value * lo, then one multiply-add with hi, is the
// quotient rounded once, so that a code is the nearest one, ties too: none of 34 million bf16 values takes another than by
// 64 bits (with one term 5294 of 17 million, with 32-bit quotients 11118 of the 34: most at exact ties). Rows of 4096 x 4096
// take 11.4 us for 11.1, 4096 x 12288 along both axes with sums 38.5 for 37.4.
struct ExactFactor {
    float hi, lo;
    __device__ __forceinline__ void divide(float amax, float largest, float inverse) {
        hi = largest / amax;
        const float rest = __builtin_fmaf(-hi, amax, largest) * (hi * inverse);   // the remainder, exact, over amax
        lo = amax < __builtin_inff() ? rest : 0.0f;                               // of infinity: hi is zero, or NaN
    }
    __device__ __forceinline__ float set(float amax, float largest, float inverse, float) {
        amax = __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, amax), kLeastBits));
        divide(amax, largest, inverse);
        return amax / largest;
    }
    __device__ __forceinline__ float operator()(float v) const { return __builtin_fmaf(v, hi, v * lo); }
};

// The same for values that have yet to be multiplied by r, a factor of their whole row: it is in the scale, and cancels in the
// codes, which so do not depend on its rounding: of 34 million normed bf16 values none takes another code than by 64 bits
// (2740 by plain 32-bit operations; 4112 x 5120 fp16 22.4 us for 22.0). Only where amax r is at the floor it does not
// cancel, and where it is NaN.
struct RowFactor : ExactFactor {
    __device__ __forceinline__ float set(float amax, float largest, float inverse, float r) {
        const float product = amax * r;
        divide(amax, largest, inverse);
        if (!(product >= kLeast)) {
            hi = product < kLeast ? largest / kLeast * r : product;
            lo = 0.0f;
        }
        return __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, product), kLeastBits)) / largest;
    }
};

// A block's scale and factor.
template <typename F>
__device__ __forceinline__ float block_scale(uint32_t amax_bits, bool e5m2, F& factor, float r = 1.0f) {
    return factor.set(__builtin_bit_cast(float, amax_bits), e5m2 ? 57344.0f : 448.0f,
                      e5m2 ? 1.0f / 57344.0f : 1.0f / 448.0f, r);
}

// Four values times factor -> four codes, the first one lowest.
template <typename F>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, F factor, bool e5m2) {
    int out = 0;
    if (e5m2) {
        out = __builtin_amdgcn_cvt_pk_bf8_f32(factor(a), factor(b), out, false);
        out = __builtin_amdgcn_cvt_pk_bf8_f32(factor(c), factor(d), out, true);
    } else {
        out = __builtin_amdgcn_cvt_pk_fp8_f32(factor(a), factor(b), out, false);
        out = __builtin_amdgcn_cvt_pk_fp8_f32(factor(c), factor(d), out, true);
    }
    return static_cast<uint32_t>(out);
}

// Where the quantized form of a matrix goes: rows of codes and block scales.
struct Quantized {
    uint8_t* codes;
    float* scale;
    int64_t ld_codes, scale_row, scale_block;
    int e5m2;
};

// q from row `row` on (null codes: left out).
inline Quantized from_row(Quantized q, int64_t row) {
    if (q.codes) {
        q.codes += row * q.ld_codes;
        q.scale += row * q.scale_row;
    }
    return q;
}

// One piece's codes. kVec: ld_codes and codes are multiples of 8, and valid is <= 0 or >= 8.
template <bool kVec, typename F>
__device__ __forceinline__ void write_codes(const Quantized& q, int64_t row, int at, int valid, const float (&v)[kPiece],
                                            F factor) {
    const u32x2v codes{codes4(v[0], v[1], v[2], v[3], factor, q.e5m2), codes4(v[4], v[5], v[6], v[7], factor, q.e5m2)};
    uint8_t* out = q.codes + row * q.ld_codes + at;
    if (valid >= kPiece) {
        if constexpr (kVec) *reinterpret_cast<u32x2v*>(out) = codes;
        else store_any(out, codes);
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
            const uint32_t word = codes[i / 4];
            if (i < valid) out[i] = static_cast<uint8_t>(word >> (8 * (i % 4)));
        }
    }
}

// One piece of a row quantized with its block's 16 lanes, all of which call this together (with valid <= 0 past the row's
// end): writes its codes, and the block's first lane the scale. r: RowFactor's.
template <bool kVec, typename F>
__device__ __forceinline__ void quantize_piece(const Quantized& q, int64_t row, int at, int valid,
                                               const float (&v)[kPiece], float r = 1.0f) {
    F factor;
    const float scale = block_scale(max16(max_bits(v)), q.e5m2, factor, r);
    if (valid <= 0) return;
    write_codes<kVec>(q, row, at, valid, v, factor);
    if (at % kBlock == 0) q.scale[row * q.scale_row + (at / kBlock) * q.scale_block] = scale;
}

// ---- host-side checks ---------------------------------------------------------------------------------------

inline bool on_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether rows of `type` with stride ld start on 16-byte boundaries (kVec also needs whole pieces: cols % 8 == 0).
inline bool rows_on_16(const void* p, int64_t ld, int type) { return on_16(p) && ld * type_bytes(type) % 16 == 0; }

constexpr int64_t kMaxSize = (int64_t{1} << 31) - 1;

// Threads of one launch. The runtime takes their number modulo 2^32 without an error (2^26 + 5 rows, four to a workgroup of
// 256 threads, wrote the first 8): more rows go in several launches.
constexpr int64_t kMaxThreads = (int64_t{1} << 32) - 1;

// A matrix that the kernels can walk: sizes under 2^31 and rows under 2 GiB, no stride under the row's length.
inline bool matrix_ok(const void* p, int64_t ld, int64_t rows, int64_t cols) {
    return p != nullptr && rows >= 1 && rows <= kMaxSize && cols >= 1 && cols <= kMaxSize / 4 && ld >= cols &&
           ld <= kMaxSize / 4;
}

inline bool type_ok(int type) { return type == FEATHER_BF16 || type == FEATHER_FP16 || type == FEATHER_FP32; }

inline bool aligned_to_type(const void* p, int type) {
    return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(type_bytes(type) - 1)) == 0;
}

// Codes and scales to write, or neither.
inline bool quantized_ok(const uint8_t* codes, int64_t ld_codes, const float* scale, int64_t rows, int64_t cols) {
    return matrix_ok(codes, ld_codes, rows, cols) && scale != nullptr && aligned_to_type(scale, FEATHER_FP32);
}

}  // namespace feather
