// The feed-forward operators' host side (include/feather_linear_ops.h): the choice of a kernel, the contract's checks and the C
// ABI, and the gated block's elementwise backward.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <iterator>

#include "feather_internal.h"
#include "feather_linear_ops.h"
#include "linear_launch.h"

namespace feather {
namespace {

constexpr int64_t kCUs = 256;
constexpr int64_t kCtrBytes = 64 * 1024;   // the workspace's arrival counters, as the other split launches'
constexpr int64_t kMaxCounters = kCtrBytes / 4;
constexpr int64_t kMaxPartBytes = kMaxSize - kCtrBytes;
constexpr int64_t kMaxDepth = int64_t{1} << 21;   // K and row strides: 256 rows of a tile stay within 31-bit offsets

int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }

bool splits_fit(const LinearPlan& plan) {
    return plan.tiles * plan.slots <= kMaxCounters && plan.tiles * plan.splits * plan.tile_bytes <= kMaxPartBytes;
}

// A tile, and microseconds: of a workgroup's start and end, and of a stage of 64 where workgroups fill the chip (per_cu on each CU)
// and where there is one alone, with what lies between in proportion; and of the join of a split K: once, of each 64 K sums that
// a tile's workgroups write and read back, and of 16 M sums in all.
struct TileCost {
    LinearKernel kernel;
    int bm, bn, per_cu;
    float fixed, full, lone;
    float join, each, all;
};
// They minimise what the pick of tile and K splits loses against the best pair, and the error of the times, in 2900 timings of 233
// shapes (100 to 4096 rows, 1024 to 28672 columns, K 512 to 14336): 1.3% in geometric mean, 31% at most; times are 10% off.
constexpr TileCost kTiles[] = {
    {kTile256, 256, 256, 1, 8.2f, 1.29f, 0.82f, 2.1f, 2.2f, 7.8f},
    {kTile256x128, 256, 128, 1, 4.4f, 0.77f, 0.41f, 2.1f, 2.2f, 7.8f},
    {kTile128, 128, 128, 2, 2.2f, 0.84f, 0.36f, 2.1f, 2.2f, 7.8f},
};
// The same of 4-bit weights, from 844 timings of 86 shapes (70 to 4096 rows): 1.1%, 14% at most; times are 8% off.
constexpr TileCost kInt4Tiles[] = {
    {kInt4Tile256, 256, 256, 1, 8.3f, 1.51f, 1.17f, 4.0f, 2.2f, 8.0f},
    {kInt4Tile128, 128, 256, 2, 4.5f, 1.88f, 0.68f, 4.0f, 2.2f, 8.0f},
};
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8};
constexpr float kLaunchCost = 2.0f;   // us from the end of one launch to the next one's work

enum class Kind { kPlain, kGated, kInt4, kInt4Gated, kInt4GatedFine };

constexpr bool is_int4(Kind kind) { return kind >= Kind::kInt4; }
constexpr bool is_gated(Kind kind) { return kind != Kind::kPlain && kind != Kind::kInt4; }

Kind int4_kind(bool gated, bool fine) { return !gated ? Kind::kInt4 : fine ? Kind::kInt4GatedFine : Kind::kInt4Gated; }

// Scales and zero points of many groups take registers that a gated kernel of 16 waves has not got: 24 rows of 5120 -> 13824 in
// groups of 32 with zero points 88 us by 2_4_4 and 54 by 2_4_2 (50 since bf16 keeps no sums of x), of 64 in bf16 50 and 43 (fp16 34 and
// 40); 1 row of 16384 -> 2048, groups of 32, 2_16_1 49, 2_8_1 33.
bool is_fine(int group, bool zeros, int type) { return zeros && (group == 32 || (group == 64 && type == FEATHER_BF16)); }

const TileCost* tiles_begin(bool int4) { return int4 ? std::begin(kInt4Tiles) : std::begin(kTiles); }
const TileCost* tiles_end(bool int4) { return int4 ? std::end(kInt4Tiles) : std::end(kTiles); }

// N: columns of b (gated: 2 F).
LinearPlan tile_plan(int64_t M, int64_t N, int64_t K, bool int4) {
    const int64_t all = ceil_div(K, 64);
    // us at 4.4 TB/s
    const float memory = (static_cast<float>(N) * (int4 ? 0.25f : 1.0f) + static_cast<float>(M)) * static_cast<float>(K) / 2.2e6f;
    LinearPlan best{};
    for (const TileCost* at = tiles_begin(int4); at != tiles_end(int4); ++at) {
        const TileCost& t = *at;
        const int64_t tiles = ceil_div(M, t.bm) * ceil_div(N, t.bn);
        const int64_t cap = kCUs * t.per_cu;
        for (const int splits : kSplits) {
            LinearPlan plan{t.kernel, splits, tiles, 256, 4, int64_t{4} * t.bm * t.bn, 0.0f};
            if (splits > 1 && (splits > all || tiles * splits > 4 * kCUs || !splits_fit(plan))) break;
            const auto stages = static_cast<float>(ceil_div(all, splits));
            const int64_t groups = tiles * splits;
            const int64_t rounds = groups / cap;
            const int64_t rest = groups - rounds * cap;
            float cost = static_cast<float>(rounds) * (stages * t.full + t.fixed);
            if (rest > 0) cost += stages * (t.lone + (t.full - t.lone) * static_cast<float>(rest) / static_cast<float>(cap)) + t.fixed;
            cost = std::max(cost, memory);
            // sums are written, and the last of a tile's workgroups reads all of its back
            if (splits > 1)
                cost += t.join + static_cast<float>(t.bm * t.bn) * static_cast<float>(splits) *
                                     (t.each / 65536.0f + static_cast<float>(tiles) * (t.all / 16777216.0f));
            plan.cost = cost + kLaunchCost;
            if (best.cost == 0.0f || plan.cost < best.cost) best = plan;
        }
    }
    return best;
}

constexpr int64_t kFewRows = 64;

// At most 64 rows, N outputs (gated: of one half). Workgroups by their columns of output; K is split over more of them where that
// still leaves `least` steps of 128 to each and no more than 256 in all.
LinearPlan few_plan(LinearKernel kernel, int rm, int rn, int wk, int wn, int64_t N, int64_t K, bool gated, int least) {
    const int64_t tiles = ceil_div(N, 16 * (gated ? rn / 2 : rn) * wn);
    LinearPlan plan{kernel, 1, tiles, 64 * wk * wn, rm * rn * wn / (gated ? 2 : 1), int64_t{1024} * rm * rn * wn, 0.0f};
    while (plan.splits < 8 && tiles * plan.splits * 2 <= kCUs && ceil_div(K, 128) / (plan.splits * 2) >= least) plan.splits *= 2;
    if (!splits_fit(plan)) plan.splits = 1;
    return plan;
}

// Measured in us, groups of 128, weights from HBM; RN_WK_WN, "/s" K splits.
//   4 bits, 1 row: 4096 x 4096 1_16_1 6.2, 1_8_1 6.9, 2_8_1 7.8; 4096 x 14336 1_16_1 11.3, 1_8_1/2 12.5; 8192 x 8192 1_8_2 12.0, 2_8_1
//   13.2, 1_16_1 16.6; 14336 x 4096 2_8_1 10.4, 2_4_2 11.5, 1_8_2 13.0. Gated, 1 row: 14336 x 4096 2_4_2 16.4, 2_8_1 19.6; 8192 x
//   8192 2_8_1 19.1, 2_4_2 20.4; 2048 x 16384 2_16_1 15.7, 2_8_1 19.8.
//   24 rows: 13824 x 5120 1_4_4 17.9, 2_4_4/2 19.3, 2_4_2 19.4; 5120 x 13824 1_4_4/2 22.2, /4 25.4, 1_8_2 26.1. Gated: 13824 x 5120
//   2_4_4 31.3, 4_4_2 31.9, 2_4_2 37.2; 4096 x 4096 2_4_2/2 11.4, 2_4_4/2 15.1.
LinearPlan int4_plan(int64_t M, int64_t N, int64_t K, bool gated, bool fine) {
    if (M > 32) return few_plan(kFew64_2_4_2, 4, 2, 4, 2, N, K, gated, 8);
    if (M > 16) {
        if (!gated) return few_plan(kFew32_1_4_4, 2, 1, 4, 4, N, K, gated, 8);
        if (N > 64 * 160 && !fine) return few_plan(kFew32_2_4_4, 2, 2, 4, 4, N, K, gated, 8);
        return few_plan(kFew32_2_4_2, 2, 2, 4, 2, N, K, gated, 8);
    }
    if (gated) {
        if (N > 8192) return few_plan(kFew16_2_4_2, 1, 2, 4, 2, N, K, gated, 16);
        if (N > 2048 || K <= 8192 || fine) return few_plan(kFew16_2_8_1, 1, 2, 8, 1, N, K, gated, 32);
        return few_plan(kFew16_2_16_1, 1, 2, 16, 1, N, K, gated, 64);
    }
    if (N > 8192) return few_plan(kFew16_2_8_1, 1, 2, 8, 1, N, K, gated, 32);
    if (N > 4096) return few_plan(kFew16_1_8_2, 1, 1, 8, 2, N, K, gated, 32);
    return few_plan(kFew16_1_16_1, 1, 1, 16, 1, N, K, gated, 64);
}

// 16-bit weights, measured alike: 1 row of 4096 -> 14336 2_8_1 42.5, 2_4_1 48.7; of 2048 -> 2048 7.5, 2_4_2 10.2; of 14336 -> 4096
// 51.4, 2_4_2 48.1. 24 rows of 5120 -> 13824 4_4_2 57.7, 2_4_2 60.4, 2_8_1 74.7.
LinearPlan gated_few_plan(int64_t M, int64_t F, int64_t K) {
    if (M > 32) return few_plan(kFew64_2_4_2, 4, 2, 4, 2, F, K, true, 8);
    if (M > 16 && F > 64 * 160) return few_plan(kFew32_4_4_2, 2, 4, 4, 2, F, K, true, 8);
    if (M > 16) return few_plan(kFew32_2_4_2, 2, 2, 4, 2, F, K, true, 8);
    if (K > 8192) return few_plan(kFew16_2_4_2, 1, 2, 4, 2, F, K, true, 8);
    return few_plan(kFew16_2_8_1, 1, 2, 8, 1, F, K, true, 16);
}

// A part of a product: rows m0 .. + M, b's columns n0 .. + N (gated: gates and ups together).
struct Part {
    int64_t m0, n0, M, N;
    LinearPlan plan;
};

struct Parts {
    Part part[4];
    int count;
    float cost;
};

// Microseconds of a launch for few rows: by its K, a workgroup's own time, or by its weights, whichever is more.
struct FewCost {
    int rows;
    float fixed, by_k, rate;
};
constexpr FewCost kInt4Few[] = {{16, 4.2f, 0.0004f, 7.1e6f}, {32, 6.9f, 0.0005f, 4.75e6f}, {64, 10.2f, 0.00066f, 2.86e6f}};
constexpr FewCost kGatedFew[] = {{16, 5.3f, 0.0011f, 2.4e6f}, {32, 9.5f, 0.00075f, 2.4e6f}, {64, 11.0f, 0.0008f, 2.05e6f}};

// One launch for a part. Few rows of a gated block or of 4-bit weights, all of the columns, go to a kernel of their own.
LinearPlan whole_plan(Kind kind, int64_t M, int64_t N, int64_t K, bool all_columns) {
    if (kind == Kind::kPlain || !all_columns || M > kFewRows) return tile_plan(M, N, K, is_int4(kind));
    const bool gated = is_gated(kind);
    LinearPlan plan = is_int4(kind) ? int4_plan(M, gated ? N / 2 : N, K, gated, kind == Kind::kInt4GatedFine)
                                    : gated_few_plan(M, N / 2, K);
    const FewCost* cost = is_int4(kind) ? kInt4Few : kGatedFew;
    while (M > cost->rows) ++cost;
    const float weights = static_cast<float>(N) * static_cast<float>(K);
    plan.cost = std::max(cost->fixed + cost->by_k * static_cast<float>(K), 2.0f + weights / cost->rate);
    return plan;
}

// Large products go in up to four launches where whole rounds of tiles end at a column or row and the rest does better on
// other tiles. Cuts fall on multiples of 256 (or on 64 rows) and are tried where a number of whole rounds of each tile ends, along either axis; a
// part may be cut once more.
Parts cut(Kind kind, int64_t m0, int64_t n0, int64_t M, int64_t N, int64_t K, bool all_columns, int depth) {
    const LinearPlan whole = whole_plan(kind, M, N, K, all_columns);
    Parts best{{{m0, n0, M, N, whole}}, 1, whole.cost};
    if (depth == 0 || whole.cost < 20.0f) return best;
    // Columns of 4-bit weights would go to tiles, which round them and want codes on 16-byte boundaries: not for few rows.
    if (is_int4(kind) && all_columns && M <= kFewRows) return best;
    const auto attempt = [&](bool rows, int64_t at) {
        const int64_t total = rows ? M : N;
        if (at <= 0 || at >= total) return;
        const LinearPlan first = rows ? whole_plan(kind, at, N, K, all_columns) : whole_plan(kind, M, at, K, false);
        if (first.cost >= best.cost) return;
        const Parts whole_heads{{{m0, n0, rows ? at : M, rows ? N : at, first}}, 1, first.cost};
        const Parts heads = depth == 1 ? whole_heads
                            : rows     ? cut(kind, m0, n0, at, N, K, all_columns, depth - 1)
                                       : cut(kind, m0, n0, M, at, K, false, depth - 1);
        const Parts rest = rows ? cut(kind, m0 + at, n0, M - at, N, K, all_columns, depth - 1)
                                : cut(kind, m0, n0 + at, M, N - at, K, false, depth - 1);
        const float cost = heads.cost + rest.cost;
        if (cost >= best.cost || heads.count + rest.count > 4) return;
        best.count = 0;
        for (int i = 0; i < heads.count; ++i) best.part[best.count++] = heads.part[i];
        for (int i = 0; i < rest.count; ++i) best.part[best.count++] = rest.part[i];
        best.cost = cost;
    };
    for (const TileCost* t = tiles_begin(is_int4(kind)); t != tiles_end(is_int4(kind)); ++t) {
        const int64_t round = kCUs * t->per_cu;
        const int64_t tiles_m = ceil_div(M, t->bm), tiles_n = ceil_div(N, t->bn);
        const int64_t rounds = tiles_m * tiles_n / round;
        if (rounds == 0) continue;
        attempt(false, rounds * round / tiles_m * t->bn / 256 * 256);
        attempt(true, rounds * round / tiles_n * t->bm / 256 * 256);
    }
    attempt(true, M / 256 * 256);
    // two launches for few rows: 96 x 4096 -> 4096 22.7 us, a tile's 27.6
    if (is_int4(kind) && M <= 2 * kFewRows) attempt(true, kFewRows);
    return best;
}

// The launches of a product: the same ones for every call of a shape. A search of large shapes takes up to 0.1 ms of the
// host, so each thread keeps the last ones by shape. Gated: N outputs, whose columns of b are whole pairs of fragments.
const Parts& parts_of(Kind kind, int64_t M, int64_t N, int64_t K) {
    struct Entry {
        Kind kind;
        int64_t M, N, K;
        Parts parts;
    };
    constexpr uint64_t kEntries = 64;
    thread_local Entry table[kEntries] = {};
    const auto hash = static_cast<uint64_t>(M) * 0x9e3779b97f4a7c15u + static_cast<uint64_t>(N) * 0xc2b2ae3d27d4eb4fu +
                      static_cast<uint64_t>(K) * 0x165667b19e3779f9u + (static_cast<uint64_t>(kind) << 36);
    Entry& e = table[(hash >> 32) % kEntries];
    if (e.M != M || e.N != N || e.K != K || e.kind != kind || e.parts.count == 0) {
        e = Entry{kind, M, N, K, cut(kind, 0, 0, M, is_gated(kind) ? 2 * ceil_div(N, 16) * 16 : N, K, true, 2)};
    }
    return e.parts;
}

int64_t workspace_of(const LinearPlan& plan) {
    return plan.splits > 1 ? kCtrBytes + plan.tiles * plan.splits * plan.tile_bytes : 0;
}

int64_t workspace_of(const Parts& parts) {
    int64_t most = 0;
    for (int i = 0; i < parts.count; ++i) most = std::max(most, workspace_of(parts.part[i].plan));
    return most;
}

// Whether each launch has fewer than 2^32 threads.
bool launchable(const LinearPlan& plan) {
    return plan.tiles * plan.splits <= kMaxThreads / plan.threads;
}

bool launchable(const Parts& parts) {
    for (int i = 0; i < parts.count; ++i)
        if (!launchable(parts.part[i].plan)) return false;
    return true;
}

// The launches of a product, one after the other.
template <typename P, typename Launch>
void launch(const P& whole, const Parts& parts, Kind kind, Launch&& go) {
    const bool gated = is_gated(kind);
    for (int i = 0; i < parts.count; ++i) {
        const Part& part = parts.part[i];
        P p = whole;
        p.splits = part.plan.splits;
        if (part.plan.kernel > kInt4Tile128) {   // all columns of the rows
            p.a += part.m0 * p.lda;
            p.c = static_cast<uint16_t*>(p.c) + part.m0 * p.ldc;
            if (p.h) p.h += part.m0 * p.ldh;
            p.M = static_cast<int32_t>(part.M);
        } else {
            const bool int4 = is_int4(kind);
            const auto tile = *std::find_if(tiles_begin(int4), tiles_end(int4),
                                            [&](const TileCost& t) { return t.kernel == part.plan.kernel; });
            p.m_first = static_cast<int32_t>(part.m0);
            p.n_first = static_cast<int32_t>(gated ? part.n0 / 2 : part.n0);
            p.tiles_m = static_cast<int32_t>(ceil_div(part.M, tile.bm));
            p.tiles_n = static_cast<int32_t>(ceil_div(part.N, tile.bn));
        }
        go(p, part.plan);
    }
}

void launch(const LinearParams& p, const Parts& parts, int type, Operands operands, hipStream_t stream) {
    const bool gated = operands == Operands::kGated || operands == Operands::kGatedKeep;
    launch(p, parts, gated ? Kind::kGated : Kind::kPlain, [&](const LinearParams& part, const LinearPlan& plan) {
        (type == FEATHER_BF16 ? linear_launch_bf16 : linear_launch_fp16)(part, plan, operands, stream);
    });
}

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
    return M >= 1 && M <= kMaxSize / 4 && N >= 1 && N <= kMaxSize / 8 && K >= 1 && K <= kMaxDepth &&
           ceil_div(M, 128) * ceil_div(N, 128) <= kMaxSize / 16;
}

bool operand_ok(const void* p, int64_t ld, int64_t cols) {
    return p && on_16(p) && ld % 8 == 0 && ld >= cols && ld <= kMaxDepth;
}

bool half_type(int type) { return type == FEATHER_BF16 || type == FEATHER_FP16; }

bool output_ok(const void* p, int64_t ld, int64_t cols, int type) {
    return p && ld >= cols && ld <= kMaxSize / 4 && aligned_to_type(p, type);
}

bool workspace_ok(const void* workspace, int64_t bytes, int64_t need) {
    return need == 0 || (workspace && bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0);
}

void use_workspace(LinearParams& p, void* workspace) {
    p.split_ctr = static_cast<uint32_t*>(workspace);
    p.split_part = workspace ? static_cast<uint8_t*>(workspace) + kCtrBytes : nullptr;
}

// ---- the gated block's elementwise backward ----
//
//   grad_gate = dy up act'(gate)     grad_up = dy act(gate)
//
// They are rounded to 16 bits as operands of the products that follow, which is what the matrix units take: the gradients of x and the
// weight are off by 2.35e-3 of their norm in bf16, of which their own rounding is 1.66e-3.
//
// A lane takes 8 columns of both halves of a few rows, whose loads are all in flight. Memory bounds it: 4096 x 12288 169 us, 4.2
// TB/s (8 rows a lane, four by four, 172; 16 178). The bias's sums are kept over more rows, 16 of them (180 us and 20 MB of sums;
// over 4 182 and 80), but 4 where 16 leave the chip without work (300 x 5504 12 us, 22).
constexpr int kThreads = 256;
constexpr int kAhead = 4;   // rows whose loads are in flight together

int rows_of(int64_t M, bool sums) { return sums && M > 512 ? 4 * kAhead : kAhead; }

struct BackwardParams {
    const uint16_t* grad_y;
    const float* kept;
    uint16_t* grad;
    float* sums;
    int64_t ld_grad_y, ld_kept, ld_grad;
    int32_t rows, cols, act, group;   // group: rows of a lane
};

template <int kType, int kAct>
__device__ __forceinline__ void backward_rows(const BackwardParams& p, int at, int valid, int row0, int row1) {
    const int half = (p.cols + 7) & ~7;
    float sum_gate[kPiece] = {}, sum_up[kPiece] = {};
    const bool last = at + kPiece >= p.cols;
    for (int first = row0; first < row1; first += kAhead) {
        RawPiece<kType> raw[kAhead];
        f32x4 gates[kAhead][2], ups[kAhead][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t row = first + i < row1 ? first + i : row1 - 1;
            const float* const kept = p.kept + row * p.ld_kept + at;
            raw[i] = load_raw<kType, false>(p.grad_y + row * p.ld_grad_y, at, valid);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                gates[i][h] = *reinterpret_cast<const f32x4*>(kept + 4 * h);
                ups[i][h] = *reinterpret_cast<const f32x4*>(kept + half + 4 * h);
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t row = first + i;
            if (row >= row1) break;
            float dy[kPiece], gate[kPiece], up[kPiece];
            unpack(raw[i], dy);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                const Slope s = activate_with_slope<kAct>(gates[i][e / 4][e % 4]);
                // the slope first: of a gate masked with the type's lowest value it is 0, and dy up may be infinite
                gate[e] = dy[e] * s.slope * ups[i][e / 4][e % 4];
                up[e] = dy[e] * s.value;
                sum_gate[e] += gate[e];
                sum_up[e] += up[e];
            }
            uint16_t* const out = p.grad + row * p.ld_grad;
            store_piece<kType, false>(out, at, valid, gate);
            store_piece<kType, false>(out + p.cols, at, valid, up);
            if (last)
                for (int c = 2 * p.cols; c < 2 * half; ++c) out[c] = 0;
        }
    }
    if (p.sums) {
        float* const out = p.sums + static_cast<int64_t>(blockIdx.y) * 2 * p.cols;
        store_piece<FEATHER_FP32, false>(out, at, valid, sum_gate);
        store_piece<FEATHER_FP32, false>(out + p.cols, at, valid, sum_up);
    }
}

template <int kType>
__global__ __launch_bounds__(kThreads) void gated_backward_kernel(const BackwardParams p) {
    const int at = static_cast<int>(blockIdx.x * kThreads + threadIdx.x) * kPiece;
    const int valid = p.cols - at;
    if (valid <= 0) return;
    const int row0 = static_cast<int>(blockIdx.y) * p.group;
    const int row1 = row0 + p.group < p.rows ? row0 + p.group : p.rows;
    if (p.act == kSilu) backward_rows<kType, kSilu>(p, at, valid, row0, row1);
    else if (p.act == kGelu) backward_rows<kType, kGelu>(p, at, valid, row0, row1);
    else backward_rows<kType, kGeluTanh>(p, at, valid, row0, row1);
}

// ---- rows put on whole lines ----

struct CopyParams {
    const uint16_t* from;
    uint16_t* to;
    int64_t ld_from, ld_to, rows;
    int32_t pieces;   // of a row
};

__global__ __launch_bounds__(kThreads) void copy_rows_kernel(const CopyParams p) {
    const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t row = index / p.pieces;
    if (row >= p.rows) return;
    const int at = static_cast<int>(index - row * p.pieces) * kPiece;
    *reinterpret_cast<u32x4*>(p.to + row * p.ld_to + at) = *reinterpret_cast<const u32x4*>(p.from + row * p.ld_from + at);
}

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" bool feather_copy_rows(const void* from, int64_t ld_from, void* to, int64_t ld_to, int64_t rows, int64_t cols,
                                  hipStream_t stream) {
    if (!matrix_ok(from, ld_from, rows, cols) || !matrix_ok(to, ld_to, rows, cols) || cols % 8 != 0 || ld_from % 8 != 0 ||
        ld_to % 8 != 0 || !on_16(from) || !on_16(to))
        return false;
    const auto pieces = static_cast<int32_t>(cols / 8);
    const int64_t most = (kMaxThreads - kThreads) / pieces;   // rows of a launch
    for (int64_t row = 0; row < rows; row += most) {
        const CopyParams p{static_cast<const uint16_t*>(from) + row * ld_from, static_cast<uint16_t*>(to) + row * ld_to, ld_from, ld_to,
                           std::min(rows - row, most), pieces};
        copy_rows_kernel<<<static_cast<uint32_t>(ceil_div(p.rows * pieces, kThreads)), kThreads, 0, stream>>>(p);
    }
    return true;
}

extern "C" int64_t feather_gated_linear_workspace_bytes(int64_t M, int64_t F, int64_t K) {
    return sizes_ok(M, 2 * F, K) ? workspace_of(parts_of(Kind::kGated, M, F, K)) : -1;
}

extern "C" bool feather_gated_linear(const void* x, int64_t ldx, const void* weight, int64_t ld_weight, const void* bias,
                                     int type, int activation, void* y, int64_t ldy, float* kept, int64_t ld_kept, int64_t M,
                                     int64_t F, int64_t K, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    const int64_t F8 = (F + 7) / 8 * 8;
    if (F < 1 || !sizes_ok(M, 2 * F, K) || K % 8 != 0 || !half_type(type) || activation < 0 || activation > 2 ||
        !operand_ok(x, ldx, K) || !operand_ok(weight, ld_weight, K) || !output_ok(y, ldy, F, type) ||
        (bias && !aligned_to_type(bias, type)))
        return false;
    if (kept && (!on_16(kept) || ld_kept % 4 != 0 || ld_kept < 2 * F8 || ld_kept >= int64_t{1} << 22)) return false;
    const Parts& parts = parts_of(Kind::kGated, M, F, K);
    const int64_t need = workspace_of(parts);
    if (!launchable(parts) || !workspace_ok(workspace, workspace_bytes, need)) return false;
    LinearParams p{};
    p.a = static_cast<const uint16_t*>(x);
    p.b = static_cast<const uint16_t*>(weight);
    p.lda = ldx;
    p.ldb = ld_weight;
    p.M = static_cast<int32_t>(M);
    p.N = static_cast<int32_t>(F);
    p.K = static_cast<int32_t>(K);
    p.bias = bias;
    p.c = y;
    p.ldc = ldy;
    p.h = kept;
    p.ldh = ld_kept;
    p.act = activation;
    use_workspace(p, need > 0 ? workspace : nullptr);
    launch(p, parts, type, kept ? Operands::kGatedKeep : Operands::kGated, stream);
    return true;
}

extern "C" int64_t feather_gated_backward_parts(int64_t M, int64_t F) {
    return M >= 1 && F >= 1 ? ceil_div(M, rows_of(M, true)) : 0;
}

extern "C" bool feather_gated_backward(const void* grad_y, int64_t ld_grad_y, const float* kept, int64_t ld_kept, int type,
                                       int activation, void* grad, int64_t ld_grad, float* sums, int64_t M, int64_t F,
                                       hipStream_t stream) {
    const int64_t F8 = (F + 7) / 8 * 8;
    if (M < 1 || M > kMaxSize || F < 1 || F > kMaxSize / 8 || !half_type(type) || activation < 0 || activation > 2 ||
        !matrix_ok(grad_y, ld_grad_y, M, F) || !aligned_to_type(grad_y, type) || !kept || !on_16(kept) || ld_kept % 4 != 0 ||
        ld_kept < 2 * F8 || !grad || !on_16(grad) || ld_grad % 8 != 0 || ld_grad < 2 * F8)
        return false;
    const int group = rows_of(M, sums != nullptr);
    constexpr int64_t kMost = 65535;   // groups of rows of a launch
    for (int64_t row = 0; row < M; row += kMost * group) {
        BackwardParams p{static_cast<const uint16_t*>(grad_y) + row * ld_grad_y, kept + row * ld_kept,
                         static_cast<uint16_t*>(grad) + row * ld_grad,
                         sums ? sums + row / group * 2 * F : nullptr, ld_grad_y, ld_kept, ld_grad,
                         static_cast<int32_t>(std::min(M - row, kMost * group)), static_cast<int32_t>(F), activation, group};
        const dim3 groups(static_cast<uint32_t>(ceil_div(F8 / 8, kThreads)), static_cast<uint32_t>(ceil_div(p.rows, group)));
        if (type == FEATHER_BF16) gated_backward_kernel<FEATHER_BF16><<<groups, kThreads, 0, stream>>>(p);
        else gated_backward_kernel<FEATHER_FP16><<<groups, kThreads, 0, stream>>>(p);
    }
    return true;
}

extern "C" int64_t feather_product_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return sizes_ok(M, N, K) ? workspace_of(parts_of(Kind::kPlain, M, N, K)) : -1;
}

extern "C" bool feather_product(const void* a, int64_t lda, bool a_across, const void* b, int64_t ldb, bool b_across,
                                const void* bias, int type, void* c, int64_t ldc, int64_t M, int64_t N, int64_t K,
                                void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (!sizes_ok(M, N, K) || !half_type(type) || (a_across && !b_across) || !operand_ok(a, lda, a_across ? M : K) ||
        !operand_ok(b, ldb, b_across ? N : K) || !output_ok(c, ldc, N, type) || (bias && !aligned_to_type(bias, type)))
        return false;
    const Parts& parts = parts_of(Kind::kPlain, M, N, K);
    const int64_t need = workspace_of(parts);
    if (!launchable(parts) || !workspace_ok(workspace, workspace_bytes, need)) return false;
    LinearParams p{};
    p.a = static_cast<const uint16_t*>(a);
    p.b = static_cast<const uint16_t*>(b);
    p.lda = lda;
    p.ldb = ldb;
    p.M = static_cast<int32_t>(M);
    p.N = static_cast<int32_t>(N);
    p.K = static_cast<int32_t>(K);
    p.bias = bias;
    p.c = c;
    p.ldc = ldc;
    use_workspace(p, need > 0 ? workspace : nullptr);
    launch(p, parts, type, a_across ? Operands::kBothAcross : b_across ? Operands::kBAcross : Operands::kAlong, stream);
    return true;
}

extern "C" int feather_linear_launches(int64_t M, int64_t N, int64_t K, bool gated, bool int4, bool fine, int64_t out[16]) {
    if (!sizes_ok(M, gated ? 2 * N : N, K)) return 0;
    const Parts& parts = parts_of(int4 ? int4_kind(gated, fine) : gated ? Kind::kGated : Kind::kPlain, M, N, K);
    for (int i = 0; i < parts.count; ++i) {
        const Part& part = parts.part[i];
        const int64_t launch[4] = {part.plan.kernel, part.plan.splits, part.M, part.N};
        std::copy(launch, launch + 4, out + 4 * i);
    }
    return parts.count;
}

// ---- 4-bit weights ----

namespace {

bool int4_ok(const uint8_t* codes, int64_t ld_codes, const void* scale, int64_t ld_scale, const uint8_t* zero, int64_t ld_zero,
             int group, int type, int64_t rows, int64_t K) {
    return codes && (reinterpret_cast<uintptr_t>(codes) & 3) == 0 && ld_codes % 4 == 0 && ld_codes >= (K + 1) / 2 &&
           ld_codes <= 2 * kMaxDepth && scale && aligned_to_type(scale, type) && ld_scale >= std::max<int64_t>(rows, 4) &&
           ld_scale <= kMaxSize && (!zero || (ld_zero >= std::max<int64_t>(rows, 4) && ld_zero <= kMaxSize)) &&
           (group == 32 || group == 64 || group == 128);
}

}  // namespace

extern "C" int64_t feather_int4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gated) {
    if (!sizes_ok(M, gated ? 2 * N : N, K)) return -1;
    const int64_t need = workspace_of(parts_of(int4_kind(gated, false), M, N, K));
    return std::max(need, workspace_of(parts_of(int4_kind(gated, true), M, N, K)));
}

extern "C" bool feather_int4_linear_direct(const uint8_t* codes, int64_t ld_codes, int64_t M, int64_t N, int64_t K, bool gated) {
    const int64_t rows = gated ? 2 * N : N;
    if (M <= kFewRows || !sizes_ok(M, rows, K)) return true;
    if (!on_16(codes) || ld_codes % 16 != 0) return false;
    // Dequantized, codes are read and values written (us at 4.4 TB/s). Of 84 shapes, 65 to 4096 rows, this picks the slower way by more
    // than 4% for four, 10% at most.
    const float before = 2.0f * kLaunchCost + static_cast<float>(rows) * static_cast<float>(K) * (2.5f / 4.4e6f);
    const float direct = parts_of(int4_kind(gated, false), M, N, K).cost;
    return direct <= before + parts_of(gated ? Kind::kGated : Kind::kPlain, M, N, K).cost;
}

extern "C" bool feather_int4_linear(const void* x, int64_t ldx, const uint8_t* codes, int64_t ld_codes, const void* scale,
                                    int64_t ld_scale, const uint8_t* zero, int64_t ld_zero, int group, const void* bias, int type,
                                    bool gated, int activation, void* y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                                    void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    const int64_t rows = gated ? 2 * N : N;
    if (N < 1 || !sizes_ok(M, rows, K) || !half_type(type) || activation < 0 || activation > 2 ||
        !operand_ok(x, ldx, K) || !output_ok(y, ldy, N, type) || (bias && !aligned_to_type(bias, type)) ||
        !int4_ok(codes, ld_codes, scale, ld_scale, zero, ld_zero, group, type, rows, K) ||
        (M > kFewRows && (!on_16(codes) || ld_codes % 16 != 0)))
        return false;
    const Kind kind = int4_kind(gated, is_fine(group, zero != nullptr, type));
    const Parts& parts = parts_of(kind, M, N, K);
    const int64_t need = workspace_of(parts);
    if (!launchable(parts) || !workspace_ok(workspace, workspace_bytes, need)) return false;
    Int4Params p{};
    p.a = static_cast<const uint16_t*>(x);
    p.lda = ldx;
    p.M = static_cast<int32_t>(M);
    p.N = static_cast<int32_t>(N);
    p.K = static_cast<int32_t>(K);
    p.bias = bias;
    p.c = y;
    p.ldc = ldy;
    p.act = activation;
    use_workspace(p, need > 0 ? workspace : nullptr);
    p.codes = codes;
    p.scale = static_cast<const uint16_t*>(scale);
    p.zero = zero;
    p.ld_codes = ld_codes;
    p.ld_scale = ld_scale;
    p.ld_zero = ld_zero;
    p.group = group;
    launch(p, parts, kind, [&](const Int4Params& part, const LinearPlan& plan) {
        (type == FEATHER_BF16 ? int4_launch_bf16 : int4_launch_fp16)(part, plan, gated, stream);
    });
    return true;
}
