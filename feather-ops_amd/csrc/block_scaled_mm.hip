// The block-scaled fp8 product's host side (include/feather_block_ops.h): the choice of a kernel, the contract's checks and
// the C ABI.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "block_mm_common.h"
#include "block_mm_launch.h"
#include "feather_internal.h"

namespace feather {
namespace {

constexpr int64_t kCUs = 256;
constexpr int64_t kCtrBytes = 64 * 1024;                // the workspace's arrival counters, as the other split launches'
constexpr int64_t kMaxCounters = kCtrBytes / 4;
constexpr int64_t kMaxPartBytes = kMaxSize - kCtrBytes;

int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }

bool splits_fit(const BlockMmPlan& plan) {
    return plan.tiles * plan.slots <= kMaxCounters && plan.tiles * plan.splits * plan.tile_bytes <= kMaxPartBytes;
}

BlockMmPlan stream_plan(BlockMmKernel kernel, int rm, int rn, int64_t M, int64_t N, int splits) {
    BlockMmPlan plan{kernel, splits, ceil_div(M, 16 * rm) * ceil_div(N, 16 * rn), rm * rn, int64_t{1024} * rm * rn, 0.0f};
    if (!splits_fit(plan)) plan.splits = 1;
    return plan;
}

// At most 64 rows. Measured (us, e4m3fn, weights from HBM; RM x RN is a workgroup's fragments, "/s" its K splits):
//   RN. A workgroup reads all rows of a beside its own rows of b, from L2: with 9 rows and more, 16 columns a workgroup read
//     as much of a as of b. 16 x 14336 x 4096: 1 x 4 14.6, 1 x 1 16.6; 16 x 4096 x 14336: 1 x 4/4 15.2, 1 x 1 16.5; 24 x
//     4096 x 14336: 2 x 4/4 16.4, 2 x 1 20.4. With one row, 1 x 1 is faster: 4096 x 14336 12.4 against 1 x 4/4 14.3; 8192 x
//     8192 14.1 against 15.7. Few columns have too few workgroups: 16 x 1024 x 4096 1 x 1/2 5.7, 1 x 4 over 7.
//   Waves. 16 take 32 blocks in flight at once, which pays where that is half of K to all of it: 1 x 4096 x 4096 5.8 against
//     6.3, 1 x 14336 x 4096 14.1 against 15.8; 1 x 4096 x 14336 13.8 against 12.4, 1 x 12288 x 2048 7.3 against 6.5.
//   Splits. Up to 256 workgroups of at least 16 blocks (8 with 17 rows and more): 1 x 1024 x 16384 /4 7.8, /2 9.0, /1 over
//     10; 1 x 1024 x 4096 /1 4.7, /2 5.1; 32 x 1024 x 4096 /4 6.4, /2 6.6.
BlockMmPlan few_rows_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t blocks = ceil_div(K, kBlock);
    const auto splits = [&](int64_t tiles, int64_t target, int64_t least) {
        int s = 1;
        while (s < 4 && tiles * s * 2 <= target && blocks / (s * 2) >= least) s *= 2;
        return s;
    };
    if (M > 32) return stream_plan(kStream4x1, 4, 1, M, N, splits(ceil_div(N, 16), 256, 8));
    const bool wide = M > 8 && (N >= 8192 || (N >= 4096 && blocks >= 64));
    if (wide) {
        const int64_t tiles = ceil_div(N, 64);
        const int s = tiles >= 192 ? 1 : splits(tiles, 512, 16);
        return M > 16 ? stream_plan(kStream2x4, 2, 4, M, N, s) : stream_plan(kStream1x4, 1, 4, M, N, s);
    }
    const int64_t tiles = ceil_div(N, 16);
    if (M > 16) return stream_plan(kStream2x1, 2, 1, M, N, splits(tiles, 256, 8));
    const BlockMmKernel kernel = blocks >= 32 && blocks <= 64 && tiles >= 256 ? kStream1x1Wide : kStream1x1;
    return stream_plan(kernel, 1, 1, M, N, splits(tiles, 256, 16));
}

// A tile of the ring kernel, and microseconds fitted to 3300 timings of 115 shapes (33 to 12288 rows, N and K 256 to 16384): a
// workgroup's start and end, and a stage with per_cu workgroups on a CU and with one. per_cu is the model's: of the 64 x 64 tile
// two fit a CU's LDS at a time (66 KiB each), and its figures for four hold what the second two wait. On the shapes of the fit
// the tile and splits with the least estimate took at most 1.12 of the best pair's time, 1.005 in geometric mean; others were
// not timed against all pairs, and large ones take more than their estimate (4096 x 14336 x 4096: 200 us, in fact 218).
struct TileCost {
    BlockMmKernel kernel;
    int bm, bn, waves, per_cu;
    float fixed, full, alone;
};
constexpr TileCost kTiles[] = {
    {kTile64x64, 64, 64, 2, 4, 2.48f, 1.578f, 0.350f},     {kTile64x128, 64, 128, 4, 2, 2.09f, 0.938f, 0.485f},
    {kTile128x128, 128, 128, 8, 1, 1.70f, 0.715f, 0.715f}, {kTile256x128, 256, 128, 8, 1, 4.43f, 0.879f, 0.879f},
    {kTile128x256, 128, 256, 8, 1, 2.78f, 1.144f, 1.144f}, {kTile256x256, 256, 256, 8, 1, 4.42f, 1.584f, 1.584f},
};
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};

BlockMmPlan tile_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t blocks = std::max<int64_t>(1, ceil_div(K, kBlock));
    const float memory = static_cast<float>(N + M) * static_cast<float>(K) / 5.0e6f;   // us at 5 TB/s
    BlockMmPlan best{};
    for (const TileCost& t : kTiles) {
        const int64_t tiles = ceil_div(M, t.bm) * ceil_div(N, t.bn);
        for (const int splits : kSplits) {
            BlockMmPlan plan{t.kernel, splits, tiles, t.waves, int64_t{4} * t.bm * t.bn, 0.0f};
            if (splits > 1 && (splits > blocks || tiles * splits > 6 * kCUs || !splits_fit(plan))) break;
            const auto stages = static_cast<float>(ceil_div(blocks, splits));
            const int64_t groups = tiles * splits;
            const int64_t rounds = groups / (kCUs * t.per_cu);
            const int64_t rest = groups - rounds * kCUs * t.per_cu;
            float cost = static_cast<float>(rounds) * (stages * t.full + t.fixed);
            if (rest > 0) {
                const float more = t.per_cu > 1 ? static_cast<float>(ceil_div(rest, kCUs) - 1) / (t.per_cu - 1) : 0.0f;
                cost += stages * (t.alone + (t.full - t.alone) * more) + t.fixed;
            }
            cost = std::max(cost, memory);
            // the last of a tile's workgroups reads all of its sums back
            if (splits > 1) cost += 0.88f + 1.44f / 65536.0f * static_cast<float>(splits * plan.tile_bytes);
            plan.cost = cost;
            if (best.cost == 0.0f || cost < best.cost) best = plan;
        }
    }
    return best;
}

// 256 rows of a tile stay within 31-bit offsets, of codes and of scales.
constexpr int64_t kMaxLd = int64_t{4} << 20;
constexpr int64_t kMaxScaleStride = int64_t{1} << 20;

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
    return M >= 1 && M <= kMaxSize / 4 && N >= 1 && N <= kMaxSize / 4 && K >= 0 && K <= kMaxLd &&
           ceil_div(M, 64) * ceil_div(N, 16) <= kMaxSize / 16;
}

// One launch for a whole product.
BlockMmPlan whole_plan(int64_t M, int64_t N, int64_t K) {
    // 33 to 64 rows stream only beside few columns: 64 x 2048 x 2048 6.5 us against 64 x 64 tiles' 7.7 and more, 64 x 4096 x
    // 4096 over 11 against 10.8.
    if (M > 64 || (M > 32 && N > 2048)) return tile_plan(M, N, K);
    BlockMmPlan plan = few_rows_plan(M, N, K);
    plan.cost = 2.0f + static_cast<float>(N) * static_cast<float>(K) / 4.5e6f;   // us: the weight at 4.5 TB/s
    return plan;
}

// A part of a product: rows m0 .. + M, columns n0 .. + N.
struct Part {
    int64_t m0, n0, M, N;
    BlockMmPlan plan;
};

struct Parts {
    Part part[4];
    int count;
    float cost;
};

constexpr float kLaunchCost = 2.0f;   // us from the end of one launch to the next one's work

// Large products go in up to four launches where whole rounds of tiles end at a column or row and the rest does better on
// other tiles: 4096 x 14336 by 256 x 256 tiles is 3.5 rounds of the 256 CUs and takes 4; 12288 columns are 3, and the other
// 2048 are one round of 128 x 256 (K = 4096: 234 us in one launch, 224 in two). Cuts fall on multiples of 256 and are
// tried where a number of whole rounds of each tile ends, along either axis; a part may be cut once more.
Parts cut(int64_t m0, int64_t n0, int64_t M, int64_t N, int64_t K, int depth) {
    const BlockMmPlan whole = whole_plan(M, N, K);
    Parts best{{{m0, n0, M, N, whole}}, 1, whole.cost};
    if (depth == 0 || whole.cost < 20.0f) return best;
    const auto attempt = [&](bool rows, int64_t at) {
        const int64_t total = rows ? M : N;
        if (at <= 0 || at >= total) return;
        const BlockMmPlan first = rows ? whole_plan(at, N, K) : whole_plan(M, at, K);
        if (first.cost + kLaunchCost >= best.cost) return;
        const Parts heads = depth > 1 ? (rows ? cut(m0, n0, at, N, K, depth - 1) : cut(m0, n0, M, at, K, depth - 1))
                                      : Parts{{{m0, n0, rows ? at : M, rows ? N : at, first}}, 1, first.cost};
        const Parts rest = rows ? cut(m0 + at, n0, M - at, N, K, depth - 1) : cut(m0, n0 + at, M, N - at, K, depth - 1);
        const float cost = heads.cost + rest.cost + kLaunchCost;
        if (cost >= best.cost || heads.count + rest.count > 4) return;
        best.count = 0;
        for (int i = 0; i < heads.count; ++i) best.part[best.count++] = heads.part[i];
        for (int i = 0; i < rest.count; ++i) best.part[best.count++] = rest.part[i];
        best.cost = cost;
    };
    for (const TileCost& t : kTiles) {
        const int64_t round = kCUs * t.per_cu;
        const int64_t tiles_m = ceil_div(M, t.bm), tiles_n = ceil_div(N, t.bn);
        const int64_t rounds = tiles_m * tiles_n / round;
        if (rounds == 0) continue;
        attempt(false, rounds * round / tiles_m * t.bn / 256 * 256);
        attempt(true, rounds * round / tiles_n * t.bm / 256 * 256);
    }
    attempt(true, M / 256 * 256);
    return best;
}

// The launches of a product: the same ones for every call of a shape. A search of large shapes takes up to 0.1 ms of the
// host, so each thread keeps the last ones by shape.
const Parts& parts_of(int64_t M, int64_t N, int64_t K) {
    struct Entry {
        int64_t M, N, K;
        Parts parts;
    };
    constexpr uint64_t kEntries = 64;
    thread_local Entry table[kEntries];
    const auto hash = static_cast<uint64_t>(M) * 0x9e3779b97f4a7c15u + static_cast<uint64_t>(N) * 0xc2b2ae3d27d4eb4fu +
                      static_cast<uint64_t>(K) * 0x165667b19e3779f9u;
    Entry& e = table[(hash >> 32) % kEntries];
    if (e.M != M || e.N != N || e.K != K || e.parts.count == 0) e = Entry{M, N, K, cut(0, 0, M, N, K, 2)};
    return e.parts;
}

int64_t workspace_bytes_of(const Parts& parts) {
    int64_t most = 0;
    for (int i = 0; i < parts.count; ++i) {
        const BlockMmPlan& plan = parts.part[i].plan;
        if (plan.splits > 1) most = std::max(most, kCtrBytes + plan.tiles * plan.splits * plan.tile_bytes);
    }
    return most;
}

// Whether each launch has fewer than 2^32 threads.
bool launchable(const Parts& parts) {
    for (int i = 0; i < parts.count; ++i) {
        const BlockMmPlan& plan = parts.part[i].plan;
        const int64_t threads = plan.kernel < kStream1x1 ? 64 * plan.slots : plan.kernel == kStream1x1Wide ? 1024 : 512;
        if (plan.tiles * plan.splits > kMaxThreads / threads) return false;   // (a tile's slots are its waves)
    }
    return true;
}

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" int64_t feather_block_scaled_mm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return sizes_ok(M, N, K) && launchable(parts_of(M, N, K)) ? workspace_bytes_of(parts_of(M, N, K)) : -1;
}

extern "C" int feather_block_scaled_mm_launches(int64_t M, int64_t N, int64_t K, int64_t out[16]) {
    if (!sizes_ok(M, N, K)) return 0;
    const Parts& parts = parts_of(M, N, K);
    for (int i = 0; i < parts.count; ++i) {
        const Part& part = parts.part[i];
        const int64_t launch[4] = {part.plan.kernel, part.plan.splits, part.M, part.N};
        std::copy(launch, launch + 4, out + 4 * i);
    }
    return parts.count;
}

extern "C" bool feather_block_scaled_mm(const uint8_t* a, int64_t lda, bool a_e5m2, const float* a_scale,
                                        int64_t a_scale_row, int64_t a_scale_block, const uint8_t* b, int64_t ldb,
                                        bool b_e5m2, const float* b_scale, int64_t b_scale_row, int64_t b_scale_block,
                                        bool b_by_row, const void* bias, void* c, int64_t ldc, int out_type, int64_t M,
                                        int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                                        hipStream_t stream) {
    if (!sizes_ok(M, N, K) || !type_ok(out_type)) return false;
    const Parts& parts = parts_of(M, N, K);
    if (!launchable(parts)) return false;
    const int64_t need = workspace_bytes_of(parts);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0))
        return false;
    if (K > 0 && (!a || !b || !a_scale || !b_scale || !on_16(a) || !on_16(b) || lda < K || ldb < K || lda % 16 != 0 ||
                  ldb % 16 != 0 || lda > kMaxLd || ldb > kMaxLd || a_scale_row < 0 || a_scale_row > kMaxScaleStride ||
                  b_scale_row < 0 || b_scale_row > kMaxScaleStride || a_scale_block < 0 || b_scale_block < 0 ||
                  !aligned_to_type(a_scale, FEATHER_FP32) || !aligned_to_type(b_scale, FEATHER_FP32)))
        return false;
    if (!c || ldc < N || ldc > kMaxSize || !aligned_to_type(c, out_type) || (bias && !aligned_to_type(bias, out_type)))
        return false;
    const int bytes = type_bytes(out_type);
    const auto launch = a_e5m2 ? (b_e5m2 ? block_mm_launch_11 : block_mm_launch_10)
                               : (b_e5m2 ? block_mm_launch_01 : block_mm_launch_00);
    for (int i = 0; i < parts.count; ++i) {
        const Part& part = parts.part[i];   // n0 is a multiple of 256: whole squares
        const BlockMmParams p{
            a + part.m0 * lda, b + part.n0 * ldb, a_scale + part.m0 * a_scale_row,
            b_scale + (b_by_row ? part.n0 : part.n0 / kBlock) * b_scale_row, lda, ldb, a_scale_row, a_scale_block,
            b_scale_row, b_scale_block, static_cast<int32_t>(part.M), static_cast<int32_t>(part.N), static_cast<int32_t>(K),
            part.plan.splits, bias ? static_cast<const uint8_t*>(bias) + part.n0 * bytes : nullptr,
            static_cast<uint8_t*>(c) + (part.m0 * ldc + part.n0) * bytes, ldc, out_type,
            static_cast<uint32_t*>(workspace), need > 0 ? static_cast<uint8_t*>(workspace) + kCtrBytes : nullptr};
        launch(p, part.plan, b_by_row, stream);
    }
    return true;
}
