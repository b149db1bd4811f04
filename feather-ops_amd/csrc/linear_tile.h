// The tile kernel of the 16-bit products, c = a b^T with either operand stored along its sum (rows of k) or across it (transposed):
// a workgroup of 4 waves owns BM x BN outputs, two waves each way, and K streams through LDS in stages of 64 that direct
// global-to-LDS loads fill.
//
// One wave a SIMD, with 256 accumulators and two halves of a stage in registers: of 256 x 256 outputs a stage takes 128 MFMAs, 32
// fragment reads and 16 loads of each wave, 223 instructions in all, laid between the MFMAs by hand. 4096 x 16384 x 4096 runs 365
// us, 1.46 PFLOP/s (the library 1.50). The matrix units are busy 79% of the clocks, at 1.94 GHz: power bounds it (operands of zeros:
// the same clocks at 2.44 GHz, 286 us). Between the loops of two tiles there are 10 us, 6 of them the outputs' way out, most of
// that memory's: all workgroups store at once.
//
// Measured, not taken: 32 x 32 x 16 MFMAs (4096 x 8192 x 4096 187 -> 215 us), outputs straight from the fragments (the same),
// non-temporal stores (27648 x 5120 x 1024 248 -> 261), starts staggered over 8 us (248 -> 246).
#pragma once

#include "linear_common.h"

namespace feather {

template <int BM_, int BN_>
struct LinearTile {
    static constexpr int BM = BM_, BN = BN_;            // 256 or 128 each
    static constexpr int kPerCu = BM + BN == 256 ? 2 : 1;   // workgroups of a CU
    static constexpr int kWaves = 4;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int RM = BM / 2 / 16;              // 16-row fragments per wave
    static constexpr int RN = BN / 2 / 16;
    static constexpr int kAUnit = BM * 128;             // bytes of an operand's stage
    static constexpr int kBUnit = BN * 128;
    // Three stages of a and two of b: a's stage t + 2 is loaded in stage t's first half, b's in its second, when every wave has
    // read b's stage t.
    static constexpr int kLdsBytes = 3 * kAUnit + 2 * kBUnit;
    static constexpr int kALoads = BM / 32;             // of a wave and stage
    static constexpr int kBLoads = BN / 32;
    static constexpr int kMfmas = RM * RN;              // of half a stage
    static constexpr int kBarrier = kMfmas / 8;         // the MFMA of the second half before which the workgroup meets
    // Fragment reads follow every kReadStep-th MFMA (past the barrier), loads are spread over the rest of their half.
    static constexpr int kReadStep = kMfmas >= 32 ? 2 : 1;
    static constexpr int kALoadStep = (kMfmas - 2) / kALoads;
    static constexpr int kBLoadStep = (kMfmas - kBarrier - 2) / kBLoads;
    static_assert((RM + RN) * kReadStep <= kMfmas - kBarrier, "a half's reads fit");
};

// 4 rows of 16 columns, transposed: of each 16 lanes, lane 4 r + c's address is row r's columns 4 c .. + 3, and lane l gets
// column l of the four rows. `restrict` gives the read an alias scope of its own: without one the compiler takes it for a reader
// of every direct load in flight and waits for them all (dx of 4096 x 24576 x 4096 1735 us).
using i16x4 = short __attribute__((ext_vector_type(4)));
using Lds16x4 = __attribute__((address_space(3))) i16x4;

__device__ __forceinline__ u32x2 read_tr16(Lds16x4* __restrict p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}

__device__ __forceinline__ u32x2 read_transposed(const uint8_t* lds, uint32_t at) {
    return read_tr16((Lds16x4*)(const_cast<uint8_t*>(lds + at)));
}

// One operand of a workgroup: where its stages come from, how they lie in LDS, and how fragments are read.
//
// Along k: rows of 64 k values, 8 pieces of 16 bytes, piece q of row r at place q ^ (r % 8), so that the 16 rows' reads of a
// piece fall on different banks. Across: rows of k, kSize columns in segments of 16 (32 bytes), segment s of row k at s ^ key(k)
// with key = k % 4 + 4 (k / 8 % 4) (% 2 for 8 segments): what a transposing read takes together, rows 8 g + r, falls on
// different banks too.
template <int kSize, bool kAcross, bool kGated>
struct Operand {
    static constexpr int kWaves = 4;
    static constexpr int R = kSize / 32;                           // fragments of a wave
    static constexpr int kKeys = kAcross && kSize == 256 ? 4 : 1;  // arrangements of a load's columns
    const uint16_t* base;      // of the workgroup's first row (or column)
    int64_t ld;
    int32_t rows, K;           // rows (columns, in whole pieces of 8) of the operand from there on, and its depth
    static constexpr int kOffsets = kAcross ? kKeys : kSize / 32;
    uint32_t off[kOffsets];    // along: of each load
    uint32_t step;             // across: between loads
    uint32_t bytes;            // along: of the workgroup's rows; across: of a stage's
    uint32_t at;               // along: of the next stage in a row
    int32_t piece;             // along: the k of this lane's piece in a stage
    uint32_t read_at;

    // first: the operand's row (column) where the workgroup starts, total: of the operand. Gated: `first` of the gates, whose
    // ups come `total` rows later; 16 rows of each in turn. part: which half of the workgroup's rows this wave reads.
    __device__ __forceinline__ void init(const uint16_t* p, int64_t ld_, int first, int total, int K_, int wave, int lane, int part) {
        ld = ld_;
        K = K_;
        const auto pitch = static_cast<uint32_t>(ld * 2);
        if constexpr (kAcross) {
            base = p + first;
            rows = (total - first + 7) & ~7;
            constexpr int kLanes = kSize / 8;                    // of a row
            const int row = 64 / kLanes * wave + lane / kLanes;   // of the first load
            const int seg = lane % kLanes / 2;
#pragma unroll
            for (int d = 0; d < kKeys; ++d) {
                const int key = kSize == 256 ? (row & 3) | d << 2 : (row & 3) | ((row >> 3) & 1) << 2;
                const int col = (seg ^ key) * 16 + (lane & 1) * 8;
                off[d] = col < rows ? static_cast<uint32_t>(row) * pitch + static_cast<uint32_t>(col) * 2u : kOob;
            }
            step = 64u / kLanes * kWaves * pitch;
            const int c = lane % 16, g = lane / 16;
            const int key = kSize == 256 ? c / 4 | g << 2 : c / 4 | (g & 1) << 2;
            read_at = static_cast<uint32_t>((8 * g + c / 4) * (kSize * 2) + ((part * R) ^ key) * 32 + c % 4 * 8);
        } else {
            const int mine = kGated && wave >= 2 ? total + first : first;   // waves 2 and 3 load the ups
            const int most = kGated ? kSize / 2 : kSize;
            base = p + mine * ld;
            rows = total - first < most ? total - first : most;
            bytes = static_cast<uint32_t>(rows - 1) * pitch + static_cast<uint32_t>((K + 7) & ~7) * 2u;
            const int row = (kGated ? 8 * (wave & 1) : 8 * wave) + lane / 8;
            const int at = (lane % 8) ^ (lane / 8);
            piece = at * 8;
#pragma unroll
            for (int d = 0; d < kOffsets; ++d)
                off[d] = static_cast<uint32_t>(row + d * (kGated ? 16 : 32)) * pitch + static_cast<uint32_t>(at) * 16u;
            const int r16 = lane % 16, g = lane / 16;
            read_at = static_cast<uint32_t>((part * 16 * R + r16) * 128 + ((g ^ (r16 % 8)) << 4));
        }
    }

    // Load d of a stage into a unit (zeros, into a unit that nobody reads, where the stage is past the end). The stage may be K's
    // last, which may have less than 64.
    __device__ __forceinline__ void load(int d, int stage, bool live, uint8_t* unit, int wave) const {
        uint8_t* const to = unit + (wave + d * kWaves) * 1024;
        if constexpr (kAcross) {
            const int left = K - stage * 64;
            const int here = left < 64 ? left : 64;
            const uint32_t size = live ? static_cast<uint32_t>(here - 1) * static_cast<uint32_t>(ld * 2) + static_cast<uint32_t>(rows) * 2u : 0u;
            dma16(make_rsrc(base + static_cast<int64_t>(stage) * 64 * ld, size), to, off[d % kKeys] + d * step);
        } else {
            dma16(make_rsrc(base, live ? bytes : 0u), to, piece < K - stage * 64 ? off[d] : kOob, static_cast<uint32_t>(stage) * 128u);
        }
    }

    // The same of whole stages, one after the other from `stage` on.
    __device__ __forceinline__ void start(int stage) {
        if constexpr (kAcross) {
            base += static_cast<int64_t>(stage) * 64 * ld;
            bytes = 63u * static_cast<uint32_t>(ld * 2) + static_cast<uint32_t>(rows) * 2u;
        } else {
            at = static_cast<uint32_t>(stage) * 128u;
        }
    }
    __device__ __forceinline__ void load_next(int d, bool live, uint8_t* lds, uint32_t unit, int wave) const {
        uint8_t* const to = lds + unit + (wave + d * kWaves) * 1024;
        const rsrc_t rsrc = make_rsrc(base, live ? bytes : 0u);
        if constexpr (kAcross) dma16(rsrc, to, off[d % kKeys] + d * step);
        else dma16(rsrc, to, off[d], at);
    }
    __device__ __forceinline__ void advance() {
        if constexpr (kAcross) base += 64 * ld;
        else at += 128;
    }

    // Fragment i of half s of a stage.
    __device__ __forceinline__ u32x4 read(const uint8_t* lds, uint32_t unit, int i, int s) const {
        if constexpr (kAcross) {
            const uint32_t at = (unit + read_at) ^ static_cast<uint32_t>(i << 5);
            const u32x2 lo = read_transposed(lds, at + s * 32 * kSize * 2);
            const u32x2 hi = read_transposed(lds, at + (s * 32 + 4) * kSize * 2);
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
            return *reinterpret_cast<const u32x4*>(lds + ((unit + read_at) ^ static_cast<uint32_t>(s << 6)) + i * 2048);
        }
    }
};

template <typename T, bool kAAcross, bool kBAcross, Form kForm, bool kBf16>
__global__ __launch_bounds__(T::kThreads) __attribute__((amdgpu_waves_per_eu(T::kPerCu, T::kPerCu)))
void linear_tile_kernel(const LinearParams p) {
    constexpr int RM = T::RM, RN = T::RN;
    constexpr bool kGated = kForm != Form::kPlain;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::kLdsBytes];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wave_m = wave / 2;
    const int wave_n = wave % 2;
    constexpr int kCols = kGated ? T::BN / 2 : T::BN;   // outputs of a tile's row
    const int tiles = p.tiles_m * p.tiles_n;
    const int split = p.splits > 1 ? static_cast<int>(blockIdx.x) / tiles : 0;
    const int tile = static_cast<int>(blockIdx.x) - split * tiles;
    int tm, tn;
    tile_of_block(tile, tiles, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = p.m_first + tm * T::BM;
    const int n0 = p.n_first + tn * kCols;
    const int all = (p.K + 63) / 64;
    const int first = static_cast<int>(static_cast<int64_t>(split) * all / p.splits);
    // The last stage comes first: the loop's loads need not look for K's end.
    const int last = static_cast<int>(static_cast<int64_t>(split + 1) * all / p.splits) - 1;
    const int stages = last + 1 - first;

    Operand<T::BM, kAAcross, false> a;
    Operand<T::BN, kBAcross, kGated> b;
    a.init(p.a, p.lda, m0, p.M, p.K, wave, lane, wave_m);
    b.init(p.b, p.ldb, n0, p.N, p.K, wave, lane, wave_n);

    f32x4 acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 x[2][RM], w[2][RN];   // of both halves of a stage

    // Units of a's stages t, t + 1 and t + 2, and of b's t and t + 1.
    uint32_t ua = 0, na = T::kAUnit, fa = 2 * T::kAUnit, ub = 3 * T::kAUnit, nb = ub + T::kBUnit;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int d = 0; d < T::kALoads; ++d) a.load(d, t ? first : last, t < stages, lds + (t ? na : ua), wave);
#pragma unroll
        for (int d = 0; d < T::kBLoads; ++d) b.load(d, t ? first : last, t < stages, lds + (t ? nb : ub), wave);
    }
    a.start(first + 1);
    b.start(first + 1);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::kALoads + T::kBLoads));
    barrier_only();
    // Read r of a half: the first row of a, the rows of b, the other rows of a, the order of their use.
    const auto read = [&](int r, int s, uint32_t unit_a, uint32_t unit_b) {
        if (r == 0) x[s][0] = a.read(lds, unit_a, 0, s);
        else if (r <= RN) w[s][r - 1] = b.read(lds, unit_b, r - 1, s);
        else if (r < RM + RN) x[s][r - RN] = a.read(lds, unit_a, r - RN, s);
    };
#pragma unroll
    for (int r = 0; r < RM + RN; ++r) read(r, 0, ua, ub);

    const auto multiply = [&](int m, int s) {
        const int i = m / RN, j = m % RN;
        acc[i][j] = mfma16<kBf16>(__builtin_bit_cast(half8, w[s][j]), __builtin_bit_cast(half8, x[s][i]), acc[i][j]);
    };
    for (int t = 0; t < stages; ++t) {
        // First half: the second half's fragments are read, a's loads of stage t + 2 issued.
#pragma unroll
        for (int m = 0; m < T::kMfmas; ++m) {
            multiply(m, 0);
            if (m % T::kReadStep == 0) read(m / T::kReadStep, 1, ua, ub);
            if (m % T::kALoadStep == 1 && m / T::kALoadStep < T::kALoads)
                a.load_next(m / T::kALoadStep, t + 2 < stages, lds, fa, wave);
            __builtin_amdgcn_sched_barrier(0);
        }
        // Second half: past the barrier stage t is read and stage t + 1 has landed, for every wave.
#pragma unroll
        for (int m = 0; m < T::kMfmas; ++m) {
            if (m == T::kBarrier) {
                __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::kALoads));
                barrier_only();
            }
            multiply(m, 1);
            if (m >= T::kBarrier) {
                const int n = m - T::kBarrier;
                if (n % T::kReadStep == 0) read(n / T::kReadStep, 0, na, nb);
                if (n % T::kBLoadStep == 1 && n / T::kBLoadStep < T::kBLoads)
                    b.load_next(n / T::kBLoadStep, t + 2 < stages, lds, ub, wave);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        a.advance();
        b.advance();
        const uint32_t freed = ua;
        ua = na;
        na = fa;
        fa = freed;
        const uint32_t other = ub;
        ub = nb;
        nb = other;
    }
    // The sums stay where they are: without this the compiler moves them about in the loop (170 copies a stage, 690 us of 590 at
    // 4096 x 24576 x 4096).
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) asm volatile("" : "+a"(acc[i][j]));
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // the last loads write LDS
    __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
    barrier_only();
    if (p.splits > 1 && !join_splits<T::kWaves>(p, acc, tile, split, wave, lane)) return;
    constexpr int kOut = OutStage<RM, kGated ? RN / 2 : RN>::kBytes;
    static_assert(T::kWaves * kOut <= T::kLdsBytes, "the epilogue's rows fit");
    finish<kForm, kBf16>(p, acc, m0 + wave_m * 16 * RM, n0 + wave_n * (kGated ? 8 : 16) * RN, lane,
                         lds + wave * kOut);
}

}  // namespace feather
