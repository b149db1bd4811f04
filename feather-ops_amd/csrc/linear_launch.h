// The kernels of the 16-bit and 4-bit products by type (linear_launch.hip, int4_launch.hip), and the launches of a product.
#pragma once

#include "int4_common.h"

namespace feather {

// Tiles by their rows and columns (kInt4Tile...: of 4-bit weights, 256 columns); kernels for few rows by their rows (kFew...), with
// RN fragments of columns a wave, WK parts of K and WN of the columns (...RN_WK_WN).
enum LinearKernel : int {
    kTile256, kTile256x128, kTile128, kInt4Tile256, kInt4Tile128,
    kFew16_1_16_1, kFew16_1_8_2, kFew16_2_8_1, kFew16_2_4_2, kFew16_2_16_1, kFew32_1_4_4, kFew32_2_4_4, kFew32_2_4_2, kFew32_4_4_2,
    kFew64_2_4_2,
};

struct LinearPlan {
    LinearKernel kernel;
    int splits;
    int64_t tiles;       // workgroups of one split
    int threads;         // of a workgroup
    int slots;           // parts of a tile that are joined by themselves
    int64_t tile_bytes;  // sums of a tile
    float cost;          // us, estimated
};

enum class Operands { kGated, kGatedKeep, kAlong, kBAcross, kBothAcross };

void linear_launch_bf16(const LinearParams& p, const LinearPlan& plan, Operands operands, hipStream_t stream);
void linear_launch_fp16(const LinearParams& p, const LinearPlan& plan, Operands operands, hipStream_t stream);

void int4_launch_bf16(const Int4Params& p, const LinearPlan& plan, bool gated, hipStream_t stream);
void int4_launch_fp16(const Int4Params& p, const LinearPlan& plan, bool gated, hipStream_t stream);

}  // namespace feather
