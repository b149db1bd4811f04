// The tile kernel of the block-scaled fp8 product: a workgroup owns BM x BN outputs, its WM x WN waves split them, and K
// streams through an LDS ring of one-block (128-deep) stages that direct global-to-LDS loads fill.
//
// A stage's 16 x 16 x 128 MFMAs take 32 clocks each and the four multiply-adds that add their result 16 of the vector unit,
// which runs beside (an MFMA stream with 4 fp32 multiply-adds an MFMA ran at 34 clocks, with 8 at 46: scales by row of b,
// which need 4 products more, are that much slower). Two waves a SIMD hide each other's LDS reads and barrier.
//
// What bounds the 256 x 256 tile, by counters at 4096 x 16384 x 4096 (235 us): the matrix units are busy 262 K of the 408 K clocks
// that a CU is (64%), a wave spends 27% of its time at waits and barriers and 31% ready but not issued, the LDS reads take 135 K
// clocks (187 bytes a clock, few conflicts); and power: the clock is 1.90 GHz on random operands and 2.36 on zeros, on which the
// same launch takes 193 us. Without the multiply-adds the product took 205 us of 235, without LDS reads 168, without the
// loads 206, without the barrier 233; as many LDS reads again for half the fragments cost 20 us. Rows of a instead of pairs, loads spread over 3 or 6 eighths of a stage, and raised wave priority
// around the MFMAs were the same or slower; 4 x 2 waves of 64 x 128 368 us.
//
// Smaller tiles have the registers to read the next stage's fragments a stage ahead (kAhead: 128 x 128 tiles 3-4% faster, 64 x
// 64 up to 8%, 64 x 128 even); they are bound by a stage's fixed costs: at 1024 x 4096 x 4096 a 128 x 128 stage took 0.69 us,
// without its loads 0.46 and without its LDS reads too 0.41, where the MFMAs alone are 0.26 by their clocks.
#pragma once

#include "block_mm_common.h"

namespace feather {

template <int BM_, int BN_, int WM_, int WN_, int kSlots_, bool kAhead_ = false, int kSpread = 5>
struct BlockTile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kSlots = kSlots_;
    static constexpr bool kAhead = kAhead_;
    static constexpr int kWaves = WM * WN;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int RM = BM / WM / 16;             // 16-row fragments of a per wave
    static constexpr int RN = BN / WN / 16;             // and of b
    static constexpr int kABytes = BM * kBlock;         // a stage: rows of 128 bytes, 16-byte pieces XOR-swizzled
    static constexpr int kBBytes = BN * kBlock;
    static constexpr int kScaleBytes = (BM + BN) * 4;   // each row's scale of the block
    static constexpr int kStageBytes = kABytes + kBBytes + kScaleBytes;
    static constexpr int kLdsBytes = kSlots * kStageBytes;
    static constexpr int kALoads = kABytes / 1024 / kWaves;
    static constexpr int kBLoads = kBBytes / 1024 / kWaves;
    static constexpr int kScaleGroups = (BM + BN) / 64; // of 64 scales
    static constexpr int kScaleLoads = (kScaleGroups + kWaves - 1) / kWaves;   // of a wave (some groups twice)
    static constexpr int kLoads = kALoads + kBLoads + kScaleLoads;
    // A stage's MFMAs go by pairs of rows, the two rows of each column one after the other, to and fro, so that one operand
    // changes from each to the next: MFMA n is row(n), col(n). Its product is added kLag MFMAs later.
    static constexpr int kMfmas = RM * RN;
    static constexpr int kPair = 2 * RN;
    static constexpr int kLag = 4;
    static constexpr int row(int n) { return n / kPair * 2 + (n + n / 2) % 2; }
    static constexpr int col(int n) { return n % kPair / 2; }
    // The pair of rows whose scales are read after MFMA n, or -1: the first at the start, the others once the pair before
    // last is done.
    static constexpr int scales_at(int n) {
        const int into = kLag < kPair ? kLag : kPair - 1;
        return n == 0 ? 0 : n % kPair == into && n / kPair + 1 < RM / 2 ? n / kPair + 1 : -1;
    }
    // The barrier that hands a slot over comes before the last pair. The refill's loads follow it, spread over kSpread / 8 of
    // a stage's MFMAs: load d after MFMA at(d), from kMfmas on in the next stage.
    static constexpr int kBarrier = kMfmas - kPair;
    static constexpr int at(int d) { return kBarrier + 1 + d * (kMfmas * kSpread / 8) / kLoads; }
    // kAhead: the barrier comes before the first MFMA, and load d after MFMA ahead_at(d) of the same stage; the next stage's
    // fragments are read in the order of their use over the stage.
    static constexpr int ahead_at(int d) { return d * kMfmas / kLoads; }
    static constexpr int kFragments = RM + RN;
    static constexpr int read_at(int f) { return f * kMfmas / kFragments; }
    static constexpr int kEarly = [] {
        int n = 0;
        while (n < kLoads && at(n) < kMfmas) ++n;
        return n;
    }();
    static_assert(at(kLoads - 1) - kMfmas < kBarrier, "a stage's loads are issued before the next barrier");
    static_assert(kMfmas >= 2 * kPair && kPair >= kLag, "two pairs of rows at least");
    static_assert(kABytes % (1024 * kWaves) == 0 && kBBytes % (1024 * kWaves) == 0, "whole loads");
    static_assert(RM % 4 == 0, "pairs of rows go through two sets of registers");
    static_assert(kBlock % (BN / WN) == 0, "a wave's columns have one square scale");
    static_assert(!kAhead || kMfmas > kLag, "scales are replaced after their last use");
    static_assert((kSlots - 1) * kLoads < 64, "vmcnt range");
};

// 4 bytes per lane straight into LDS.
__device__ __forceinline__ void dma4(rsrc_t r, const uint8_t* lds_dst, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (__attribute__((address_space(3))) void*)(reinterpret_cast<uintptr_t>(lds_dst)), 4, static_cast<int>(voff), 0,
        0, 0);
}

// The epilogue: a wave's 16 RN-column outputs, 16 rows at a time through LDS of its own, so that a row leaves as whole
// pieces of 8 outputs on neighbouring lanes (of any alignment: 4096 x 5001 x 2576 took 76 us value by value, with 5000
// columns 65).
template <int RN>
struct OutRow {
    static constexpr int kCols = 16 * RN;
    static constexpr int kPitch = kCols + 4;    // floats: the 16 rows' writes of a column fall on different banks
};

template <int kType, int RM, int RN>
__device__ __forceinline__ void store_typed(const BlockMmParams& p, const f32x4 (&acc)[RM][RN], int row0, int col0,
                                            int lane, float* own) {
    using O = OutRow<RN>;
    constexpr int kLanes = O::kCols / kPiece;   // of a row
    const int r16 = lane % 16;
    const int g = lane / 16;
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
        for (int j = 0; j < RN; ++j) *reinterpret_cast<f32x4*>(own + r16 * O::kPitch + 16 * j + 4 * g) = acc[i][j];
        __builtin_amdgcn_s_waitcnt(kLgkm0Imm);   // a wave's LDS operations are done in order
#pragma unroll
        for (int at = 0; at < 16 * kLanes; at += 64) {
            const int r = (at + lane) / kLanes;
            const int c = (at + lane) % kLanes * kPiece;
            const int m = row0 + 16 * i + r;
            const int n = col0 + c;
            if (m >= p.M || n >= p.N || r >= 16) continue;
            const float* from = own + r * O::kPitch + c;
            float v[kPiece];
#pragma unroll
            for (int e = 0; e < kPiece; ++e) v[e] = from[e];
            if (p.bias) {
                float add[kPiece];
                load_piece<kType, false>(p.bias, n, p.N - n, add);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) v[e] += add[e];
            }
            store_piece<kType, false>(static_cast<uint8_t*>(p.c) + static_cast<int64_t>(m) * p.ldc * type_bytes(kType), n,
                                      p.N - n, v);
        }
        __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
    }
}

template <int RM, int RN>
__device__ __forceinline__ void store_tile(const BlockMmParams& p, const f32x4 (&acc)[RM][RN], int row0, int col0, int lane,
                                           float* own) {
    if (p.out_type == FEATHER_BF16) store_typed<FEATHER_BF16>(p, acc, row0, col0, lane, own);
    else if (p.out_type == FEATHER_FP16) store_typed<FEATHER_FP16>(p, acc, row0, col0, lane, own);
    else store_typed<FEATHER_FP32>(p, acc, row0, col0, lane, own);
}

template <typename T, bool kAE5M2, bool kBE5M2, bool kByRow>
__global__ __launch_bounds__(T::kThreads) void block_tile_kernel(const BlockMmParams p) {
    constexpr int RM = T::RM, RN = T::RN;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::kLdsBytes];
    const int tid = threadIdx.x;
    const int lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wave_m = wave / T::WN;
    const int wave_n = wave % T::WN;
    const int tiles_m = (p.M + T::BM - 1) / T::BM;
    const int tiles_n = (p.N + T::BN - 1) / T::BN;
    // Workgroup -> (K range, tile), ranges of one tile a whole round of tiles apart.
    const int tiles = tiles_m * tiles_n;
    const int split = p.splits > 1 ? static_cast<int>(blockIdx.x) / tiles : 0;
    const int tile = static_cast<int>(blockIdx.x) - split * tiles;
    int tm, tn;
    tile_of_block(tile, tiles, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::BM;
    const int n0 = tn * T::BN;
    const int blocks = (p.K + kBlock - 1) / kBlock;
    const int first = static_cast<int>(static_cast<int64_t>(split) * blocks / p.splits);
    const int stages = static_cast<int>(static_cast<int64_t>(split + 1) * blocks / p.splits) - first;
    const bool tail = p.K % 16 != 0 && first + stages == blocks;   // the last block ends inside a 16-byte piece

    // Direct loads: each fills 8 rows of 8 pieces; lane l's place is piece l % 8 of row l / 8, which holds the row's piece
    // (l % 8) ^ (row % 8), so that 8 rows' reads of one piece fall on 8 different places.
    const rsrc_t a_rsrc = rows_rsrc(p.a, p.lda, m0, p.M, T::BM, p.K);
    const rsrc_t b_rsrc = rows_rsrc(p.b, p.ldb, n0, p.N, T::BN, p.K);
    const rsrc_t null_rsrc = make_rsrc(p.a, 0u);
    const int piece_at = ((lane % 8) ^ (lane / 8)) * 16;
    const uint32_t a_off = static_cast<uint32_t>(wave * 8 + lane / 8) * static_cast<uint32_t>(p.lda) + piece_at;
    const uint32_t b_off = static_cast<uint32_t>(wave * 8 + lane / 8) * static_cast<uint32_t>(p.ldb) + piece_at;
    const uint32_t a_step = 8u * T::kWaves * static_cast<uint32_t>(p.lda);
    const uint32_t b_step = 8u * T::kWaves * static_cast<uint32_t>(p.ldb);
    // This wave's groups of 64 scales of a stage.
    uint32_t scale_off[T::kScaleLoads];
    const float* scale_base[T::kScaleLoads];
    int64_t scale_step[T::kScaleLoads];
    int scale_group[T::kScaleLoads];
#pragma unroll
    for (int s = 0; s < T::kScaleLoads; ++s) {
        const int group = (wave + s * T::kWaves) % T::kScaleGroups;
        const bool of_a = group < T::BM / 64;
        const int row = (of_a ? m0 : n0 - T::BM) + group * 64 + lane;
        const int64_t base = of_a ? m0 : kByRow ? n0 : n0 / kBlock;
        const int64_t index = of_a || kByRow ? row : row / kBlock;
        const int64_t pitch = of_a ? p.as_row : p.bs_row;
        scale_group[s] = group;
        scale_off[s] = row < (of_a ? p.M : p.N) ? static_cast<uint32_t>((index - base) * pitch) * 4u : kOob;
        scale_base[s] = (of_a ? p.a_scale : p.b_scale) + base * pitch;
        scale_step[s] = of_a ? p.as_block : p.bs_block;
    }

    // Load d of stage `at` (past the last: nothing, into a slot nobody reads).
    const auto load = [&](int d, int at, uint32_t slot) {
        const bool live = at < stages;
        const int kb = first + at;
        uint8_t* const stage = lds + slot;
        if (d < T::kALoads + T::kBLoads) {
            const bool is_a = d < T::kALoads;
            const int i = is_a ? d : d - T::kALoads;
            const uint32_t off = is_a ? a_off + i * a_step : b_off + i * b_step;
            const bool there = piece_at < p.K - kb * kBlock;
            dma16(live ? (is_a ? a_rsrc : b_rsrc) : null_rsrc, stage + (is_a ? 0 : T::kABytes) + (wave + i * T::kWaves) * 1024,
                  there ? off : kOob, static_cast<uint32_t>(kb) * kBlock);
        } else {
            const int i = d - T::kALoads - T::kBLoads;
            dma4(make_rsrc(scale_base[i] + kb * scale_step[i], live ? 0x7fffffffu : 0u),
                 stage + T::kABytes + T::kBBytes + scale_group[i] * 256, scale_off[i]);
        }
    };
    // The last stage's bytes past K (K % 16 != 0: inside a 16-byte piece) become zero.
    const auto clear_tail = [&](uint32_t slot) {
        const int piece = p.K % kBlock / 16;
        for (int r = tid; r < T::BM + T::BN; r += T::kThreads) {
            auto* at = reinterpret_cast<u32x4*>(lds + slot + r * kBlock + ((piece ^ (r % 8)) << 4));
            *at = keep_bytes(*at, p.K % 16);
        }
        __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
        barrier_only();
    };

    const int g = lane / 16;
    const int r16 = lane % 16;
    const uint32_t a_rd = static_cast<uint32_t>((wave_m * 16 * RM + r16) * kBlock + ((g ^ (r16 % 8)) << 4));
    const uint32_t b_rd = static_cast<uint32_t>(T::kABytes + (wave_n * 16 * RN + r16) * kBlock + ((g ^ (r16 % 8)) << 4));
    const uint32_t sa_rd = static_cast<uint32_t>(T::kABytes + T::kBBytes + (wave_m * 16 * RM + r16) * 4);
    const uint32_t sb_rd = static_cast<uint32_t>(T::kABytes + T::kBBytes + (T::BM + wave_n * 16 * RN) * 4);
    // Fragment i of a row block: pieces g and g + 4, whose places differ in one bit.
    const auto read_fragment = [&](uint32_t slot, uint32_t rd, int i) {
        return join16(*reinterpret_cast<const u32x4*>(lds + slot + rd + i * 2048),
                      *reinterpret_cast<const u32x4*>(lds + slot + (rd ^ 64u) + i * 2048));
    };
    using ScaleB = std::conditional_t<kByRow, f32x4, float>;
    constexpr int kScalesB = kByRow ? RN : 1;
    static_assert(T::kWaves * 16 * OutRow<RN>::kPitch * 4 <= T::kLdsBytes, "the epilogue's rows fit");

    f32x4 acc[RM][RN], t[T::kLag];
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
        for (int i = 0; i < RM; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < T::kLag; ++n) t[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (T::kAhead) {
        i32x8 fa[2][RM], fb[2][RN];     // of a stage and the next
        float sa[2][RM];
        ScaleB sb[2][kScalesB];
#pragma unroll
        for (int i = 0; i < RM; ++i) sa[1][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < kScalesB; ++j) sb[1][j] = ScaleB{};
        // Fragment f of a stage in the order of its use: two rows of a, the columns of b, the other rows.
        const auto read = [&](auto set, uint32_t slot, int f) {
            constexpr int s = set();
            if (f < 2) fa[s][f] = read_fragment(slot, a_rd, f);
            else if (f < 2 + RN) fb[s][f - 2] = read_fragment(slot, b_rd, f - 2);
            else fa[s][f - RN] = read_fragment(slot, a_rd, f - RN);
        };
        const auto read_scales = [&](auto set, uint32_t slot) {
            constexpr int s = set();
#pragma unroll
            for (int i = 0; i < RM; ++i) sa[s][i] = *reinterpret_cast<const float*>(lds + slot + sa_rd + i * 64);
#pragma unroll
            for (int j = 0; j < kScalesB; ++j) {
                if constexpr (kByRow) sb[s][j] = *reinterpret_cast<const f32x4*>(lds + slot + sb_rd + j * 64 + g * 16);
                else sb[s][j] = *reinterpret_cast<const float*>(lds + slot + sb_rd);
            }
        };
        using Even = std::integral_constant<int, 0>;
        using Odd = std::integral_constant<int, 1>;

#pragma unroll
        for (int s = 0; s < T::kSlots; ++s)
#pragma unroll
            for (int d = 0; d < T::kLoads; ++d) load(d, s, s * T::kStageBytes);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((T::kSlots - 1) * T::kLoads));
        barrier_only();
        if (tail && stages == 1) clear_tail(0);
#pragma unroll
        for (int f = 0; f < T::kFragments; ++f) read(Even{}, 0, f);
        read_scales(Even{}, 0);

        uint32_t cur = 0;
        const auto stage = [&](int kb, auto set, auto other) {
            const uint32_t nxt = cur + T::kStageBytes == T::kLdsBytes ? 0 : cur + T::kStageBytes;
            // This stage is in registers, and the next has landed, for every wave past the barrier: the slot is free.
            __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
            __builtin_amdgcn_s_waitcnt(vmcnt_imm((T::kSlots - 2) * T::kLoads));
            barrier_only();
            if (tail && kb + 2 == stages) clear_tail(nxt);
#pragma unroll
            for (int n = 0; n < T::kMfmas; ++n) {
                const int i = T::row(n), j = T::col(n);
                const int before = (n + T::kMfmas - T::kLag) % T::kMfmas;
                const int bi = T::row(before), bj = T::col(before);
                constexpr int s = set(), o = other();
                f32x4& sum = acc[bi][bj];
                if (n < T::kLag) add_scaled(sum, t[n % T::kLag], sa[o][bi] * sb[o][kByRow ? bj : 0]);
                else add_scaled(sum, t[n % T::kLag], sa[s][bi] * sb[s][kByRow ? bj : 0]);
                asm volatile("" : "+v"(sum));   // as below: in place, not behind the MFMAs
                t[n % T::kLag] = mfma_block<kAE5M2, kBE5M2>(fb[s][j], fa[s][i]);
#pragma unroll
                for (int f = 0; f < T::kFragments; ++f)
                    if (T::read_at(f) == n) read(other, nxt, f);
                if (n == T::kLag) read_scales(other, nxt);
#pragma unroll
                for (int d = 0; d < T::kLoads; ++d)
                    if (T::ahead_at(d) == n) load(d, kb + T::kSlots, cur);
                __builtin_amdgcn_sched_barrier(0);
            }
            cur = nxt;
        };
        for (int kb = 0; kb < stages; kb += 2) {
            stage(kb, Even{}, Odd{});
            if (kb + 1 < stages) stage(kb + 1, Odd{}, Even{});
        }
        const auto last = [&](auto set) {
            constexpr int kFirst = T::kMfmas - T::kLag;
            constexpr int s = set();
#pragma unroll
            for (int n = 0; n < T::kLag; ++n) {
                const int i = T::row(kFirst + n), j = T::col(kFirst + n);
                add_scaled(acc[i][j], t[(kFirst + n) % T::kLag], sa[s][i] * sb[s][kByRow ? j : 0]);
            }
        };
        if (stages % 2 == 0) last(Odd{});
        else last(Even{});
    } else {
        i32x8 fa[2][2], fb[RN];     // two pairs of rows of a
        float sa[2][2];             // of two pairs of rows
        ScaleB sb[kScalesB], sb_next{};
        sa[1][0] = sa[1][1] = 0.0f;
#pragma unroll
        for (int j = 0; j < kScalesB; ++j) sb[j] = ScaleB{};

#pragma unroll
        for (int s = 0; s < T::kSlots; ++s)
#pragma unroll
            for (int d = 0; d < (s + 1 < T::kSlots ? T::kLoads : T::kEarly); ++d) load(d, s, s * T::kStageBytes);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((T::kSlots - 2) * T::kLoads + T::kEarly));
        barrier_only();
        if (tail && stages == 1) clear_tail(0);
#pragma unroll
        for (int j = 0; j < RN; ++j) fb[j] = read_fragment(0, b_rd, j);
        fa[0][0] = read_fragment(0, a_rd, 0);
        fa[0][1] = read_fragment(0, a_rd, 1);

        uint32_t cur = 0;
        uint32_t prv = (T::kSlots - 1) * T::kStageBytes;
        const auto stage = [&](int kb, auto may_end) {
            const uint32_t nxt = cur + T::kStageBytes == T::kLdsBytes ? 0 : cur + T::kStageBytes;
#pragma unroll
            for (int n = 0; n < T::kMfmas; ++n) {
                const int i = T::row(n), j = T::col(n);
                {
                    // The product of kLag MFMAs ago (at first: of the stage before, with its scales) leaves its registers to this
                    // one's. The empty asm keeps the compiler from gathering the multiply-adds behind the stage's MFMAs, where
                    // nothing hides them.
                    const int before = (n + T::kMfmas - T::kLag) % T::kMfmas;
                    const int bi = T::row(before), bj = T::col(before);
                    f32x4& sum = acc[bi][bj];
                    add_scaled(sum, t[n % T::kLag], sa[bi / 2 % 2][bi % 2] * sb[kByRow ? bj : 0]);
                    asm volatile("" : "+v"(sum));
                }
                if (n == T::kBarrier) {
                    // All of this stage's operands are read and the next stage has landed, for every wave past the barrier.
                    __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
                    __builtin_amdgcn_s_waitcnt(vmcnt_imm((T::kSlots - 2) * T::kLoads));
                    barrier_only();
                    if (may_end() && kb + 2 == stages) clear_tail(nxt);
                }
                t[n % T::kLag] = mfma_block<kAE5M2, kBE5M2>(fb[j], fa[i / 2 % 2][i % 2]);
                // Operands: a pair of rows during the pair before, a column of b after its last use.
                const int q = n % T::kPair;
                const int next_row = n / T::kPair * 2 + 2;
                if (q < 2) {
                    fa[next_row / 2 % 2][q] = next_row < RM ? read_fragment(cur, a_rd, next_row + q) : read_fragment(nxt, a_rd, q);
                }
                if (n >= T::kBarrier && n % 2 == 1) fb[j] = read_fragment(nxt, b_rd, j);
                // Scales, ahead of their first use, behind the last one of what they replace and, being the stage's, ahead of its
                // barrier; those of b in the first pair.
                const int pair = T::scales_at(n);
                if (pair >= 0) {
                    sa[pair % 2][0] = *reinterpret_cast<const float*>(lds + cur + sa_rd + pair * 128);
                    sa[pair % 2][1] = *reinterpret_cast<const float*>(lds + cur + sa_rd + pair * 128 + 64);
                }
                if constexpr (kByRow) {
#pragma unroll
                    for (int c = 0; c < RN; ++c)
                        if (n == (2 * c + 1 + T::kLag < T::kPair ? 0 : T::kLag - 1))
                            sb[c] = *reinterpret_cast<const f32x4*>(lds + cur + sb_rd + c * 64 + g * 16);
                } else {
                    if (n == 0) sb_next = *reinterpret_cast<const float*>(lds + cur + sb_rd);
                    if (n == T::kLag - 1) sb[0] = sb_next;
                }
#pragma unroll
                for (int d = 0; d < T::kLoads; ++d) {
                    if (T::at(d) == n) load(d, kb + T::kSlots, cur);
                    if (T::at(d) - T::kMfmas == n) load(d, kb + T::kSlots - 1, prv);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            prv = cur;
            cur = nxt;
        };
        const int plain = !tail ? stages : stages < 2 ? 0 : stages - 2;
        int kb = 0;
        for (; kb < plain; ++kb) stage(kb, std::false_type{});
        for (; kb < stages; ++kb) stage(kb, std::true_type{});
#pragma unroll
        for (int n = 0; n < T::kLag; ++n) {
            constexpr int kFirst = T::kMfmas - T::kLag;
            const int i = T::row(kFirst + n), j = T::col(kFirst + n);
            add_scaled(acc[i][j], t[(kFirst + n) % T::kLag], sa[i / 2 % 2][i % 2] * sb[kByRow ? j : 0]);
        }
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // the last loads write LDS
    __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
    barrier_only();
    if (p.splits > 1 && !join_splits<T::kWaves, RM, RN>(p, acc, tile, split, wave, lane)) return;
    store_tile<RM, RN>(p, acc, m0 + wave_m * 16 * RM, n0 + wave_n * 16 * RN, lane,
                       reinterpret_cast<float*>(lds + wave * (16 * OutRow<RN>::kPitch * 4)));
}

}  // namespace feather
