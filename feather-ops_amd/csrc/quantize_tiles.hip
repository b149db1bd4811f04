// A matrix quantized to blocks of 128 along its rows, along its columns (stored transposed) or in squares of 128 x 128,
// from one reading (include/feather_block_ops.h): what training a layer in fp8 needs of its activations, weights and
// gradients, and what loading a weight needs.
//
// A workgroup takes one 128 x 128 tile: 16 lanes to a row's block as everywhere, and each value's bits into LDS, where a
// lane then walks two neighbouring columns over 32 rows (one LDS word a row, lanes on consecutive words: no conflicts).
// The four waves' quarters of a column meet in LDS for its largest value and its sum, in wave order; its codes pass through
// LDS once more to leave as whole lines.
//
// Memory bounds it, once the transposed stores are whole lines: bf16 4096 x 12288 in both directions 42.7 us, 4.8 TB/s, as
// squares in both 38.4 (58 with scattered stores and branching loads).
#include <hip/hip_runtime.h>

#include <algorithm>
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
};

template <int kType, bool kVec, bool kSquare>
__global__ __launch_bounds__(kThreads) void tiles_kernel(const TilesParams p) {
    using Raw = RawPiece<kType>;
    constexpr int kWord = kType == FEATHER_FP32 ? 2 : 1;   // dwords of two neighbouring values
    __shared__ __attribute__((aligned(16))) uint32_t values[kBlock][kBlock / 2 * kWord];
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

    Raw raw[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int r = s * 16 + tid / 16;
        const int64_t row = row0 + (r < rows ? r : rows - 1);
        const int from = r < rows ? at : p.cols;   // past the last row: what lies past its end, nothing
        raw[s] = load_raw<kType, kVec>(static_cast<const uint8_t*>(p.x) + row * p.ldx * type_bytes(kType), from, p.cols - from);
    }
    uint32_t most = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int r = s * 16 + tid / 16;
        if (walk) {
            auto* to = reinterpret_cast<u32x4v*>(&values[r][tid % 16 * (kPiece / 2) * kWord]);
#pragma unroll
            for (int h = 0; h < Raw::kWords / 4; ++h)
                to[h] = u32x4v{raw[s].w[4 * h], raw[s].w[4 * h + 1], raw[s].w[4 * h + 2], raw[s].w[4 * h + 3]};
        }
        float v[kPiece];
        unpack(raw[s], v);
        if constexpr (kSquare) {
            most = max(most, max_bits(v));
        } else {
            // valid <= 0 past the last row: quantize_piece writes nothing there
            if (p.q.codes) quantize_piece<kVec, ExactFactor>(p.q, row0 + r, at, r < rows ? p.cols - at : 0, v);
        }
    }
    ExactFactor factor{};
    float scale = 0.0f;
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
                float v[kPiece];
                unpack(raw[s], v);
                write_codes<kVec>(p.q, row0 + r, at, r < rows ? p.cols - at : 0, v, factor);
            }
        }
    }
    if (!walk) return;

    // Columns 2 lane and 2 lane + 1, rows 32 wave .. + 31; rows past the end hold zeros.
    float w[2][kWalk], sum[2] = {0.0f, 0.0f};
    uint32_t col_most[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kWalk; ++i) {
        const uint32_t* word = &values[wave * kWalk + i][lane * kWord];
        if constexpr (kType == FEATHER_FP32) {
            w[0][i] = __builtin_bit_cast(float, word[0]);
            w[1][i] = __builtin_bit_cast(float, word[1]);
        } else {
            w[0][i] = to_float<kType>(word[0] & 0xffffu);
            w[1][i] = to_float<kType>(word[0] >> 16);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            col_most[c] = max(col_most[c], abs_bits(w[c][i]));
            sum[c] += w[c][i];
        }
    }
    __syncthreads();   // joint_max[.][0] of the square's largest value, and the values, have been read
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        joint_max[wave][2 * lane + c] = col_most[c];
        joint_sum[wave][2 * lane + c] = sum[c];
    }
    __syncthreads();
    // The transposed codes go to LDS, over the values: a column's 128 bytes as 8 pieces of 16, XOR-swizzled by the column, so
    // that they leave as whole lines, 8 lanes to a column.
    auto* staged = reinterpret_cast<u32x4v*>(&values[0][0]);
    static_assert(sizeof(values) >= kBlock * kBlock, "a tile's codes fit over its values");
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int j = 2 * lane + c;
        const int col = col0 + j;
        if (p.sums && wave == 0 && col < p.cols)
            p.sums[tile_m * p.cols + col] = (joint_sum[0][j] + joint_sum[1][j]) + (joint_sum[2][j] + joint_sum[3][j]);
        if (!p.t.codes) continue;
        if constexpr (!kSquare) {
            scale = block_scale(max(max(joint_max[0][j], joint_max[1][j]), max(joint_max[2][j], joint_max[3][j])),
                                p.t.e5m2, factor);
            if (wave == 0 && col < p.cols) p.t.scale[col * p.t.scale_row + tile_m * p.t.scale_block] = scale;
        }
#pragma unroll
        for (int h = 0; h < kWalk / 16; ++h) {
            const float* x = &w[c][16 * h];
            staged[j * 8 + ((wave * (kWalk / 16) + h) ^ (j / 2 % 8))] =
                u32x4v{codes4(x[0], x[1], x[2], x[3], factor, p.t.e5m2), codes4(x[4], x[5], x[6], x[7], factor, p.t.e5m2),
                       codes4(x[8], x[9], x[10], x[11], factor, p.t.e5m2),
                       codes4(x[12], x[13], x[14], x[15], factor, p.t.e5m2)};
        }
    }
    if (!p.t.codes) return;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kBlock * kBlock / 16 / kThreads; ++s) {
        const int j = (s * kThreads + tid) / 8;
        const int piece = tid % 8;
        const int valid = rows - 16 * piece;
        if (col0 + j >= p.cols || valid <= 0) continue;
        const u32x4v codes = staged[j * 8 + (piece ^ (j / 2 % 8))];
        uint8_t* out = p.t.codes + (col0 + j) * p.t.ld_codes + row0 + 16 * piece;
        if (valid >= 16) {
            store_any(out, codes);   // ld_codes_t is any
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t word = codes[i / 4];
                if (i < valid) out[i] = static_cast<uint8_t>(word >> (8 * (i % 4)));
            }
        }
    }
}

// p from row of tiles `tile` on.
TilesParams from_tile(TilesParams p, int64_t tile, int type, bool square) {
    const int64_t row = tile * kBlock;
    p.x = static_cast<const uint8_t*>(p.x) + row * p.ldx * type_bytes(type);
    if (p.q.codes) {
        p.q.codes += row * p.q.ld_codes;
        p.q.scale += (square ? tile : row) * p.q.scale_row;
    }
    if (p.t.codes) {
        p.t.codes += row;
        p.t.scale += tile * p.t.scale_block;
    }
    if (p.sums) p.sums += tile * p.cols;
    p.rows -= row;
    return p;
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
    const TilesParams p{x, {codes, scale, ld_codes, scale_row, scale_block, e5m2},
                        {codes_t, scale_t, ld_codes_t, scale_t_row, scale_t_block, e5m2}, sums, ldx, rows,
                        static_cast<int32_t>(cols), static_cast<int32_t>(tiles_n)};
    const bool vec = cols % kPiece == 0 && rows_on_16(x, ldx, type) && (!codes || (on_16(codes) && ld_codes % 8 == 0));
    const int64_t tiles_m = (rows + kBlock - 1) / kBlock;
    const int64_t most = kMaxThreads / kThreads / tiles_n;   // rows of tiles of a launch
    const auto go = [&](auto t, auto v) {
        for (int64_t tile = 0; tile < tiles_m; tile += most) {
            const TilesParams part = from_tile(p, tile, type, square);
            const auto grid = static_cast<uint32_t>(std::min(tiles_m - tile, most) * tiles_n);
            if (square) tiles_kernel<t(), v(), true><<<grid, kThreads, 0, stream>>>(part);
            else tiles_kernel<t(), v(), false><<<grid, kThreads, 0, stream>>>(part);
        }
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
