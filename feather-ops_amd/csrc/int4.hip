// 4-bit weights: their quantization, and back to 16 bits (include/feather_linear_ops.h). Streams through memory, which bounds the way
// back: 14336 x 4096 to 16 bits 26-34 us, 4.3-5.6 TB/s, of which the values written are four fifths. Quantizing it takes 43-54 us a call, once
// a weight.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "feather_linear_ops.h"
#include "int4_common.h"

namespace feather {
namespace {

constexpr int kThreads = 256;

struct WeightParams {
    const void* w;
    uint8_t* codes;
    void* scale;
    uint8_t* zero;
    int64_t ldw, ld_codes, ld_scale, ld_zero, rows;
    int32_t K, group, pieces;   // pieces of 8 columns of a row, whole groups
};

template <int kLanes>
__device__ __forceinline__ float across(float v, bool largest) {
#pragma unroll
    for (int by = 1; by < kLanes; by *= 2) {
        const float other = __shfl_xor(v, by);
        v = largest ? fmaxf(v, other) : fminf(v, other);
    }
    return v;
}

// A lane takes a piece of 8 columns, kLanes of them a group, whose first one writes the scale. Pieces are counted over all rows.
template <int kType, int kLanes>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const WeightParams p) {
    const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t row = index / p.pieces;
    if (row >= p.rows) return;   // whole groups of lanes: a row's pieces are a multiple of kLanes
    const int at = static_cast<int>(index - row * p.pieces) * kPiece;
    const int valid = p.K - at;
    float v[kPiece];
    load_piece<kType, false>(static_cast<const uint8_t*>(p.w) + row * p.ldw * type_bytes(kType), at, valid, v);
    float low = 0.0f, high = 0.0f;
    uint32_t most = max_bits(v);
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
        low = fminf(low, v[e]);
        high = fmaxf(high, v[e]);
    }
#pragma unroll
    for (int by = 1; by < kLanes; by *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), by)));
    float scale, zero = 8.0f;
    if (p.zero) {
        low = across<kLanes>(low, false);
        high = across<kLanes>(high, true);
        const float range = high - low;
        scale = range < __builtin_huge_valf() ? range / 15.0f : high / 15.0f - low / 15.0f;   // past fp32's range
    } else {
        scale = __builtin_bit_cast(float, most) / 7.0f;
    }
    const bool finite = most < 0x7f800000u;
    if (!finite) scale = __builtin_bit_cast(float, most);
    const uint32_t bits = to_bits<kType>(scale);
    scale = to_float<kType>(bits);
    const bool usable = finite && scale > 0.0f;
    if (p.zero && usable) zero = fminf(fmaxf(rintf(-low / scale), 0.0f), 15.0f);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
        const float q = usable && e < valid ? fminf(fmaxf(rintf(v[e] / scale) + zero, 0.0f), 15.0f) : zero;
        word |= static_cast<uint32_t>(q) << (4 * e);
    }
    // rows can be written up to a multiple of 4 bytes
    if (valid > 0) *reinterpret_cast<uint32_t*>(p.codes + row * p.ld_codes + at / 2) = word;
    if (at % (kLanes * kPiece) == 0) {
        const int64_t g = at / (kLanes * kPiece);
        static_cast<uint16_t*>(p.scale)[g * p.ld_scale + row] = static_cast<uint16_t>(bits);
        if (p.zero) p.zero[g * p.ld_zero + row] = static_cast<uint8_t>(zero);
    }
}

// A lane takes 8 codes.
template <int kType>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const WeightParams p) {
    const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t row = index / p.pieces;
    if (row >= p.rows) return;
    const int at = static_cast<int>(index - row * p.pieces) * kPiece;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(p.codes + row * p.ld_codes + at / 2);
    const int g = at / p.group;
    const float scale = to_float<kType>(static_cast<const uint16_t*>(p.scale)[g * p.ld_scale + row]);
    const float zero = p.zero ? static_cast<float>(p.zero[g * p.ld_zero + row]) : 8.0f;
    float v[kPiece];
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
        v[e] = at + e < p.K ? (static_cast<float>(word >> (4 * e) & 15u) - zero) * scale : 0.0f;
    store_piece<kType, true>(static_cast<uint8_t*>(const_cast<void*>(p.w)) + row * p.ldw * type_bytes(kType), at, kPiece, v);
}

// p from row `row` on.
WeightParams from_row(WeightParams p, int64_t row) {
    p.w = static_cast<const uint8_t*>(p.w) + row * p.ldw * 2;
    p.codes += row * p.ld_codes;
    p.scale = static_cast<uint16_t*>(p.scale) + row;
    if (p.zero) p.zero += row;
    p.rows -= row;
    return p;
}

template <typename Launch>
void by_rows(const WeightParams& p, Launch launch) {
    const int64_t most = (kMaxThreads - kThreads) / p.pieces;   // rows of a launch
    for (int64_t row = 0; row < p.rows; row += most) {
        WeightParams part = from_row(p, row);
        part.rows = std::min(part.rows, most);
        launch(part, static_cast<uint32_t>((part.rows * p.pieces + kThreads - 1) / kThreads));
    }
}

bool weight_ok(const WeightParams& p, int type) {
    const int64_t bytes = (int64_t{p.K} + 7) / 8 * 4;   // whole dwords of codes
    return (type == FEATHER_BF16 || type == FEATHER_FP16) && (p.group == 32 || p.group == 64 || p.group == 128) &&
           matrix_ok(p.w, p.ldw, p.rows, p.K) && p.codes && (reinterpret_cast<uintptr_t>(p.codes) & 3) == 0 &&
           p.ld_codes % 4 == 0 && p.ld_codes >= bytes && p.ld_codes <= kMaxSize && p.scale && aligned_to_type(p.scale, type) &&
           p.ld_scale >= p.rows && p.ld_scale <= kMaxSize && (!p.zero || (p.ld_zero >= p.rows && p.ld_zero <= kMaxSize)) &&
           aligned_to_type(p.w, type);
}

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" bool feather_int4_quantize(const void* w, int64_t ldw, int type, int group, uint8_t* codes, int64_t ld_codes,
                                      void* scale, int64_t ld_scale, uint8_t* zero, int64_t ld_zero, int64_t N, int64_t K,
                                      hipStream_t stream) {
    if (K < 1 || K > kMaxSize / 4) return false;
    const WeightParams p{w, codes, scale, zero, ldw, ld_codes, ld_scale, ld_zero, N, static_cast<int32_t>(K), group,
                         group > 0 ? static_cast<int32_t>((K + group - 1) / group * (group / kPiece)) : 0};
    if (!weight_ok(p, type)) return false;
    by_rows(p, [&](const WeightParams& part, uint32_t groups) {
        const auto go = [&](auto t) {
            if (group == 32) quantize_kernel<t(), 4><<<groups, kThreads, 0, stream>>>(part);
            else if (group == 64) quantize_kernel<t(), 8><<<groups, kThreads, 0, stream>>>(part);
            else quantize_kernel<t(), 16><<<groups, kThreads, 0, stream>>>(part);
        };
        if (type == FEATHER_BF16) go(std::integral_constant<int, FEATHER_BF16>{});
        else go(std::integral_constant<int, FEATHER_FP16>{});
    });
    return true;
}

extern "C" bool feather_int4_dequantize(const uint8_t* codes, int64_t ld_codes, const void* scale, int64_t ld_scale,
                                        const uint8_t* zero, int64_t ld_zero, int group, int type, void* w, int64_t ldw, int64_t N,
                                        int64_t K, hipStream_t stream) {
    if (K < 1 || K > kMaxSize / 4) return false;
    const WeightParams p{w, const_cast<uint8_t*>(codes), const_cast<void*>(scale), const_cast<uint8_t*>(zero), ldw, ld_codes,
                         ld_scale, ld_zero, N, static_cast<int32_t>(K), group, static_cast<int32_t>((K + 7) / 8)};
    if (!weight_ok(p, type) || !on_16(w) || ldw % 8 != 0) return false;
    by_rows(p, [&](const WeightParams& part, uint32_t groups) {
        if (type == FEATHER_BF16) dequantize_kernel<FEATHER_BF16><<<groups, kThreads, 0, stream>>>(part);
        else dequantize_kernel<FEATHER_FP16><<<groups, kThreads, 0, stream>>>(part);
    });
    return true;
}
