// Which kernel a block-scaled fp8 product runs on, and the launchers, one translation unit per pair of fp8 formats
// (block_mm_launch.hip).
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace feather {

struct BlockMmParams;

// The kernels: tiles of the ring kernel (block_mm_tile.h), then the streaming kernel's shapes (block_mm_stream.h) by the
// fragments of 16 x 16 outputs a workgroup has along M and N.
enum BlockMmKernel {
    kTile64x64,
    kTile64x128,
    kTile128x128,
    kTile128x256,
    kTile256x128,
    kTile256x256,
    kStream1x1,
    kStream1x1Wide,   // 16 waves
    kStream1x4,
    kStream2x1,
    kStream2x4,
    kStream4x1,
};

struct BlockMmPlan {
    BlockMmKernel kernel;
    int splits;             // K ranges, joined in the workspace
    int64_t tiles, slots;   // output tiles, and the parts of one that are joined by themselves
    int64_t tile_bytes;     // of a tile's fp32 sums
    float cost;             // estimated microseconds
};

void block_mm_launch_00(const BlockMmParams& p, const BlockMmPlan& plan, bool by_row, hipStream_t stream);
void block_mm_launch_01(const BlockMmParams& p, const BlockMmPlan& plan, bool by_row, hipStream_t stream);
void block_mm_launch_10(const BlockMmParams& p, const BlockMmPlan& plan, bool by_row, hipStream_t stream);
void block_mm_launch_11(const BlockMmParams& p, const BlockMmPlan& plan, bool by_row, hipStream_t stream);

}  // namespace feather
