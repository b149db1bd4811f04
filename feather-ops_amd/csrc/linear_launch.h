// The kernels of the 16-bit and 4-bit products by type (linear_launch.hip, int4_launch.hip), and the launches of a product.
#pragma once

#include "int4_common.h"

namespace feather {

enum LinearKernel : int { kTile256, kTile256x128, kTile128, kFewRows16, kFewRows32, kFewRows64 };

struct LinearPlan {
    LinearKernel kernel;
    int splits;
    int64_t tiles;       // workgroups of one split
    int slots;           // parts of a tile that are joined by themselves
    int64_t tile_bytes;  // sums of a tile
    float cost;          // us, estimated
};

enum class Operands { kGated, kGatedKeep, kAlong, kBAcross, kBothAcross };

void linear_launch_bf16(const LinearParams& p, const LinearPlan& plan, Operands operands, hipStream_t stream);
void linear_launch_fp16(const LinearParams& p, const LinearPlan& plan, Operands operands, hipStream_t stream);

void int4_launch_bf16(const Int4Params& p, const LinearPlan& plan, bool gated, hipStream_t stream);
void int4_launch_fp16(const Int4Params& p, const LinearPlan& plan, bool gated, hipStream_t stream);

// Columns of a workgroup of the few-rows kernels.
constexpr int few_rows_columns(bool gated) { return gated ? 16 : 32; }

}  // namespace feather
