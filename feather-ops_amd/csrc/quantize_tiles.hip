// A matrix quantized to blocks of 128 along its rows, along its columns (stored transposed) or in squares of 128 x 128,
// from one reading (include/feather_block_ops.h): what training a layer in fp8 needs of its activations, weights and
// gradients, and what loading a weight needs.
//
// A workgroup takes one 128 x 128 tile: 16 lanes to a row's block as everywhere, and each value's bits into LDS, where a
// lane then walks two neighbouring columns over 32 rows (one LDS word a row, lanes on consecutive words: no conflicts).
// The four waves' quarters of a column meet in LDS for its largest value and its sum, in wave order.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "block_common.h"

namespace feather {
namespace {

constexpr int kThreads = 256;
constexpr int kSteps = kBlock * kBlock / kPiece / kThreads;   // pieces of a tile per lane: 8
constexpr int kWalk = kBlock / 4;                             // rows of a column per lane: 32

struct TilesParams {
    const void* x;
    Quantized q, t;         // null codes: left out
    float* sums;            // null: left out
    int64_t ldx, rows;
    int32_t cols, tiles_n;
    int32_t t_on_16;        // rows of the transposed codes start on 16-byte boundaries
};

template <int kType, bool kVec, bool kSquare>
__global__ __launch_bounds__(kThreads) void tiles_kernel(const TilesParams p) {
    using Word = std::conditional_t<kType == FEATHER_FP32, u32x2v, uint32_t>;   // two neighbouring values
    __shared__ __attribute__((aligned(16))) Word values[kBlock][kBlock / 2];
    __shared__ uint32_t joint_max[4][kBlock];
    __shared__ float joint_sum[4][kBlock];
    const int tid = threadIdx.x;
    const int lane = tid % 64;
    const int wave = tid / 64;
    const int64_t tile_m = blockIdx.x / p.tiles_n;
    const int tile_n = static_cast<int>(blockIdx.x - tile_m * p.tiles_n);
    const int64_t row0 = tile_m * kBlock;
    const int col0 = tile_n * kBlock;
    const int rows = p.rows - row0 < kBlock ? static_cast<int>(p.rows - row0) : kBlock;
    const int at = col0 + tid % 16 * kPiece;
    const bool walk = p.t.codes || p.sums;

    float v[kSteps][kPiece];
    uint32_t most = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int r = s * 16 + tid / 16;
        const int valid = r < rows ? p.cols - at : 0;
        load_piece<kType, kVec>(static_cast<const uint8_t*>(p.x) + (row0 + r) * p.ldx * type_bytes(kType), at, valid, v[s]);
        if constexpr (kSquare) most = max(most, max_bits(v[s]));
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int r = s * 16 + tid / 16;
        if (walk) {
            auto* to = &values[r][tid % 16 * (kPiece / 2)];
#pragma unroll
            for (int i = 0; i < kPiece / 2; ++i) {
                if constexpr (kType == FEATHER_FP32) {
                    to[i] = u32x2v{to_bits<kType>(v[s][2 * i]), to_bits<kType>(v[s][2 * i + 1])};
                } else {
                    to[i] = pack2<kType>(v[s][2 * i], v[s][2 * i + 1]);
                }
            }
        }
        if constexpr (!kSquare) {
            // valid <= 0 past the last row: quantize_piece writes nothing there
            if (p.q.codes) quantize_piece<kVec>(p.q, row0 + r, at, r < rows ? p.cols - at : 0, v[s]);
        }
    }
    float factor = 0.0f, scale = 0.0f;
    if constexpr (kSquare) {
        most = max16(most);
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
        if (lane == 0) joint_max[wave][0] = most;
    }
    __syncthreads();
    if constexpr (kSquare) {
        most = max(max(joint_max[0][0], joint_max[1][0]), max(joint_max[2][0], joint_max[3][0]));
        scale = block_scale(most, p.q.e5m2, factor);
        if (tid == 0) {
            if (p.q.codes) p.q.scale[tile_m * p.q.scale_row + tile_n * p.q.scale_block] = scale;
            if (p.t.codes) p.t.scale[tile_n * p.t.scale_row + tile_m * p.t.scale_block] = scale;
        }
        if (p.q.codes) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int r = s * 16 + tid / 16;
                const int valid = r < rows ? p.cols - at : 0;
                uint8_t* out = p.q.codes + (row0 + r) * p.q.ld_codes + at;
                const u32x2v codes{codes4(v[s][0], v[s][1], v[s][2], v[s][3], factor, p.q.e5m2),
                                   codes4(v[s][4], v[s][5], v[s][6], v[s][7], factor, p.q.e5m2)};
                if (kVec && valid >= kPiece) {
                    *reinterpret_cast<u32x2v*>(out) = codes;
                } else {
#pragma unroll
                    for (int i = 0; i < kPiece; ++i) {
                        const uint32_t word = codes[i / 4];
                        if (i < valid) out[i] = static_cast<uint8_t>(word >> (8 * (i % 4)));
                    }
                }
            }
        }
    }
    if (!walk) return;

    // Columns 2 lane and 2 lane + 1, rows 32 wave .. + 31; rows past the end hold zeros.
    float w[2][kWalk], sum[2] = {0.0f, 0.0f};
    uint32_t col_most[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kWalk; ++i) {
        const Word word = values[wave * kWalk + i][lane];
        if constexpr (kType == FEATHER_FP32) {
            const uint32_t x0 = word[0], x1 = word[1];
            w[0][i] = __builtin_bit_cast(float, x0);
            w[1][i] = __builtin_bit_cast(float, x1);
        } else {
            w[0][i] = to_float<kType>(word & 0xffffu);
            w[1][i] = to_float<kType>(word >> 16);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            col_most[c] = max(col_most[c], abs_bits(w[c][i]));
            sum[c] += w[c][i];
        }
    }
    __syncthreads();   // joint_max[.][0] of the square's largest value has been read
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        joint_max[wave][2 * lane + c] = col_most[c];
        joint_sum[wave][2 * lane + c] = sum[c];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int j = 2 * lane + c;
        const int col = col0 + j;
        if (col >= p.cols) continue;
        if (p.sums && wave == 0)
            p.sums[tile_m * p.cols + col] = (joint_sum[0][j] + joint_sum[1][j]) + (joint_sum[2][j] + joint_sum[3][j]);
        if (!p.t.codes) continue;
        if constexpr (!kSquare) {
            scale = block_scale(max(max(joint_max[0][j], joint_max[1][j]), max(joint_max[2][j], joint_max[3][j])),
                                p.t.e5m2, factor);
            if (wave == 0) p.t.scale[col * p.t.scale_row + tile_m * p.t.scale_block] = scale;
        }
        uint32_t codes[kWalk / 4];
#pragma unroll
        for (int i = 0; i < kWalk / 4; ++i)
            codes[i] = codes4(w[c][4 * i], w[c][4 * i + 1], w[c][4 * i + 2], w[c][4 * i + 3], factor, p.t.e5m2);
        const int valid = rows - wave * kWalk;
        uint8_t* out = p.t.codes + col * p.t.ld_codes + row0 + wave * kWalk;
        if (p.t_on_16 && valid >= kWalk) {
#pragma unroll
            for (int i = 0; i < kWalk / 16; ++i)
                reinterpret_cast<u32x4v*>(out)[i] =
                    u32x4v{codes[4 * i], codes[4 * i + 1], codes[4 * i + 2], codes[4 * i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < kWalk; ++i)
                if (i < valid) out[i] = static_cast<uint8_t>(codes[i / 4] >> (8 * (i % 4)));
        }
    }
}

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" bool feather_quantize_tiles(const void* x, int type, int64_t ldx, bool square, uint8_t* codes,
                                       int64_t ld_codes, float* scale, int64_t scale_row, int64_t scale_block,
                                       uint8_t* codes_t, int64_t ld_codes_t, float* scale_t, int64_t scale_t_row,
                                       int64_t scale_t_block, float* sums, bool e5m2, int64_t rows, int64_t cols,
                                       hipStream_t stream) {
    if (!type_ok(type) || !matrix_ok(x, ldx, rows, cols) || !aligned_to_type(x, type)) return false;
    if ((codes == nullptr) != (scale == nullptr) || (codes_t == nullptr) != (scale_t == nullptr)) return false;
    if (codes && !quantized_ok(codes, ld_codes, scale, rows, cols)) return false;
    if (codes_t && (rows > kMaxSize / 4 || !quantized_ok(codes_t, ld_codes_t, scale_t, cols, rows))) return false;
    if (!codes && !codes_t && !sums) return false;
    const int64_t tiles_n = (cols + kBlock - 1) / kBlock;
    const int64_t tiles = tiles_n * ((rows + kBlock - 1) / kBlock);
    if (tiles > kMaxSize) return false;
    const TilesParams p{x, {codes, scale, ld_codes, scale_row, scale_block, e5m2},
                        {codes_t, scale_t, ld_codes_t, scale_t_row, scale_t_block, e5m2}, sums, ldx, rows,
                        static_cast<int32_t>(cols), static_cast<int32_t>(tiles_n), on_16(codes_t) && ld_codes_t % 16 == 0};
    const bool vec = rows_on_16(x, ldx, type) && (!codes || (on_16(codes) && ld_codes % 8 == 0));
    const auto grid = static_cast<uint32_t>(tiles);
    const auto go = [&](auto t, auto v) {
        if (square) tiles_kernel<t(), v(), true><<<grid, kThreads, 0, stream>>>(p);
        else tiles_kernel<t(), v(), false><<<grid, kThreads, 0, stream>>>(p);
    };
    const auto typed = [&](auto t) {
        if (vec) go(t, std::true_type{});
        else go(t, std::false_type{});
    };
    if (type == FEATHER_BF16) typed(std::integral_constant<int, FEATHER_BF16>{});
    else if (type == FEATHER_FP16) typed(std::integral_constant<int, FEATHER_FP16>{});
    else typed(std::integral_constant<int, FEATHER_FP32>{});
    return true;
}
