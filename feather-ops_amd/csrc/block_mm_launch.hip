// The block-scaled fp8 product's kernels for one pair of formats: FEATHER_A_E5M2 and FEATHER_B_E5M2 are 0 (e4m3fn) or 1.
#include "block_mm_launch.h"
#include "block_mm_stream.h"
#include "block_mm_tile.h"

namespace feather {
namespace {

constexpr bool kA = FEATHER_A_E5M2 != 0;
constexpr bool kB = FEATHER_B_E5M2 != 0;

uint32_t ceil_div(int32_t x, int y) { return static_cast<uint32_t>((static_cast<int64_t>(x) + y - 1) / y); }

template <typename T>
void tile(const BlockMmParams& p, bool by_row, hipStream_t stream) {
    const uint32_t grid = ceil_div(p.M, T::BM) * ceil_div(p.N, T::BN) * static_cast<uint32_t>(p.splits);
    if (by_row) block_tile_kernel<T, kA, kB, true><<<grid, T::kThreads, 0, stream>>>(p);
    else block_tile_kernel<T, kA, kB, false><<<grid, T::kThreads, 0, stream>>>(p);
}

template <typename T>
void stream_rows(const BlockMmParams& p, bool by_row, hipStream_t stream) {
    const dim3 grid(ceil_div(p.N, 16 * T::RN), ceil_div(p.M, 16 * T::RM), static_cast<uint32_t>(p.splits));
    if (by_row) block_stream_kernel<T, kA, kB, true><<<grid, T::kThreads, 0, stream>>>(p);
    else block_stream_kernel<T, kA, kB, false><<<grid, T::kThreads, 0, stream>>>(p);
}

}  // namespace

#define FEATHER_CAT_(a, b, c) a##b##c
#define FEATHER_CAT(a, b, c) FEATHER_CAT_(a, b, c)

void FEATHER_CAT(block_mm_launch_, FEATHER_A_E5M2, FEATHER_B_E5M2)(const BlockMmParams& p, const BlockMmPlan& plan,
                                                                    bool by_row, hipStream_t stream) {
    switch (plan.kernel) {
        case kTile64x64: tile<BlockTile<64, 64, 1, 2, 4, true>>(p, by_row, stream); break;
        case kTile64x128: tile<BlockTile<64, 128, 1, 4, 3, true>>(p, by_row, stream); break;
        case kTile128x128: tile<BlockTile<128, 128, 2, 4, 3, true>>(p, by_row, stream); break;
        case kTile128x256: tile<BlockTile<128, 256, 2, 4, 3>>(p, by_row, stream); break;
        case kTile256x128: tile<BlockTile<256, 128, 4, 2, 3>>(p, by_row, stream); break;
        case kTile256x256: tile<BlockTile<256, 256, 2, 4, 2>>(p, by_row, stream); break;
        case kStream1x1: stream_rows<BlockStream<1, 1, 8, 2>>(p, by_row, stream); break;
        case kStream1x1Wide: stream_rows<BlockStream<1, 1, 16, 2>>(p, by_row, stream); break;
        case kStream1x4: stream_rows<BlockStream<1, 4, 8, 1>>(p, by_row, stream); break;
        case kStream2x1: stream_rows<BlockStream<2, 1, 8, 2>>(p, by_row, stream); break;
        case kStream2x4: stream_rows<BlockStream<2, 4, 8, 2>>(p, by_row, stream); break;
        case kStream4x1: stream_rows<BlockStream<4, 1, 8, 2>>(p, by_row, stream); break;
    }
}

}  // namespace feather
