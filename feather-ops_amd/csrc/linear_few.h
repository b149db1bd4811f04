// The kernel for few rows, with 16-bit or 4-bit weights. The weight is read once, straight into registers, and that is what
// bounds it; the rows of x, which every workgroup reads, go through LDS. One row of 4096 -> 14336 gated takes 44 us in 16 bits (5.3
// TB/s) and with 4-bit weights 16.4 in fp16 and 16.8 in bf16 (3.7; the loads alone 14.5), 24 rows of 5120 -> 13824 57 and 32.5 (5.0 and 2.3; the loads alone
// 25: codes become 16 bits between them).
//
// A workgroup's waves are WK parts of K by WN parts of its columns. An iteration takes WK steps of 128 k's, one to each part: its
// rows of x are in one of two LDS buffers, in the order in which the matrix instructions take them, the next iteration's on
// their way to the other one by registers, the weights an iteration ahead in registers. (Rows of x straight into registers held
// up the weights: loads come back in order.)
#pragma once

#include "int4_common.h"

namespace feather {

// RM x RN 16 x 16 fragments a wave (gated: RN / 2 of gates and as many of ups).
template <int RM_, int RN_, int WK_, int WN_>
struct FewRows {
    static constexpr int RM = RM_, RN = RN_, WK = WK_, WN = WN_;
    static constexpr int kWaves = WK * WN;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int kRows = 16 * RM;
    static constexpr int kStepBytes = kRows * 256;         // a step's rows
    static constexpr int kBufferBytes = WK * kStepBytes;
    static constexpr int kJoinBytes = kWaves * RM * RN * 1024;
    static constexpr int kLdsBytes = 2 * kBufferBytes > kJoinBytes ? 2 * kBufferBytes : kJoinBytes;
    static constexpr int kPieces = kRows * 16 / (64 * WN);   // 16-byte pieces of x of a thread and iteration
    static_assert(kRows * 16 % (64 * WN) == 0, "whole pieces");
};

constexpr int kStep = 128;

// Four outputs of row m at columns n .. n + 3.
template <bool kBf16>
__device__ __forceinline__ void store4(const LinearParams& p, int m, int n, f32x4 v) {
    uint16_t* const out = static_cast<uint16_t*>(p.c) + static_cast<int64_t>(m) * p.ldc + n;
    const int valid = p.N - n;
    constexpr int kType = kTypeOf<kBf16>;
    if (valid >= 4) {
        store_any(out, u32x2{pack2<kType>(v[0], v[1]), pack2<kType>(v[2], v[3])});
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < valid) out[e] = static_cast<uint16_t>(to_bits<kType>(v[e]));
    }
}

// A row's sums, in units of `unit`, to outputs: gate and up of columns n .. n + 3, or (plain) the sums themselves.
template <Form kForm, bool kBf16>
__device__ __forceinline__ void store_sums(const LinearParams& p, int m, int n, f32x4 sum, f32x4 up, float unit) {
    if (m >= p.M || n >= p.N) return;
    sum = sum * unit + bias4<kBf16>(p.bias, n, p.N);
    if constexpr (kForm != Form::kPlain) {
        up = up * unit + bias4<kBf16>(p.bias, int64_t{p.N} + n, int64_t{2} * p.N);
        if constexpr (kForm == Form::kGatedKeep) {
            float* const row = p.h + static_cast<int64_t>(m) * p.ldh + n;   // both halves padded to 8 columns
            store_any(row, sum);
            store_any(row + ((p.N + 7) & ~7), up);
        }
        if (p.act == kSilu) sum = gate4<kSilu>(sum, up);
        else if (p.act == kGelu) sum = gate4<kGelu>(sum, up);
        else sum = gate4<kGeluTanh>(sum, up);
    }
    store4<kBf16>(p, m, n, sum);
}

// kGroups: a step's groups of 4-bit codes (4, 2 or 1 of 32, 64 or 128), or 0: 16-bit weights. kZeros: the codes have zero points
// of their own.
template <typename T, int kGroups, bool kZeros, Form kForm, bool kBf16>
__global__ __launch_bounds__(T::kThreads) void few_rows_kernel(const std::conditional_t<kGroups != 0, Int4Params, LinearParams> p) {
    constexpr bool kInt4 = kGroups != 0;
    constexpr int RM = T::RM, RN = T::RN, WK = T::WK, WN = T::WN;
    constexpr bool kGated = kForm != Form::kPlain;
    static_assert(!kGated || RN % 2 == 0, "gates and ups go in pairs");
    constexpr int kWaveCols = 16 * (kGated ? RN / 2 : RN);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::kLdsBytes];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int part = wave / WN;
    const int n0 = static_cast<int>(blockIdx.x) * (kWaveCols * WN) + wave % WN * kWaveCols;
    const int split = static_cast<int>(blockIdx.y);
    const int r16 = lane % 16;
    const int g = lane / 16;
    const int all = (p.K + kStep - 1) / kStep;
    const int first = static_cast<int>(static_cast<int64_t>(split) * all / p.splits);
    const int end = static_cast<int>(static_cast<int64_t>(split + 1) * all / p.splits);
    const int turns = (end - first + WK - 1) / WK;
    const int k_end = end * kStep < p.K ? end * kStep : p.K;

    // ---- rows of x ----
    //
    // A lane's k's of a step: 8 of each MFMA, 32 s + 8 g; of 4-bit groups of 128, which one lane may hold any part of, 32 g + 8 s, as
    // its 16 bytes of codes have them (other groups' dwords change lanes first). 4-bit: in the codes' order.
    constexpr bool kRun = kGroups == 1;
    constexpr int kTurnPieces = 16 * WK;   // of a row
    u32x4 piece[T::kPieces];
    const auto load_rows = [&](int turn) {
#pragma unroll
        for (int i = 0; i < T::kPieces; ++i) {
            const int q = i * T::kThreads + static_cast<int>(threadIdx.x);
            const int row = q / kTurnPieces;
            const int k = (first + turn * WK) * kStep + q % kTurnPieces * 8;
            piece[i] = u32x4{0u, 0u, 0u, 0u};
            if (row < p.M && k < k_end) piece[i] = *reinterpret_cast<const u32x4*>(p.a + row * p.lda + k);
        }
    };
    const auto write_rows = [&](int turn) {
        uint8_t* const to = lds + (turn & 1) * T::kBufferBytes;
#pragma unroll
        for (int i = 0; i < T::kPieces; ++i) {
            const int q = i * T::kThreads + static_cast<int>(threadIdx.x);
            const int row = q / kTurnPieces;
            const int at = q % kTurnPieces;
            const int s = kRun ? at % 4 : at / 4 % 4;
            const int c = kRun ? at / 4 % 4 : at % 4;
            u32x4 v = piece[i];
            if constexpr (kInt4) v = __builtin_bit_cast(u32x4, order8<kBf16>(v));
            if (row < p.M) *reinterpret_cast<u32x4*>(to + at / 16 * T::kStepBytes + (s * T::kRows + row) * 64 + c * 16) = v;
        }
    };
    const uint32_t x_at = static_cast<uint32_t>(part * T::kStepBytes + r16 * 64 + g * 16);
    const auto read_rows = [&](int turn, int s, int i) {
        return *reinterpret_cast<const u32x4*>(lds + (turn & 1) * T::kBufferBytes + x_at + (s * T::kRows + 16 * i) * 64);
    };

    // ---- weights: fragment j is 16 rows from row_of(j) ----
    const auto row_of = [&](int j) { return kGated ? 16 * (j / 2) : 16 * j; };
    const int here = p.N - n0 < kWaveCols ? p.N - n0 : kWaveCols;   // may be none
    const uint8_t* weight;
    int64_t pitch;
    if constexpr (kInt4) {
        weight = p.codes;
        pitch = p.ld_codes;
    } else {
        weight = reinterpret_cast<const uint8_t*>(p.b);
        pitch = p.ldb * 2;
    }
    const int row_bytes = kInt4 ? ((p.K + 1) / 2 + 3) & ~3 : ((p.K + 7) & ~7) * 2;
    const uint32_t records = here > 0 ? static_cast<uint32_t>(here - 1) * static_cast<uint32_t>(pitch) + static_cast<uint32_t>(row_bytes) : 0u;
    const rsrc_t w_rsrc[2] = {make_rsrc(weight + n0 * pitch, records),
                              make_rsrc(weight + (kGated ? p.N + static_cast<int64_t>(n0) : n0) * pitch, records)};
    const uint32_t w_off = static_cast<uint32_t>(r16) * static_cast<uint32_t>(pitch) + 16u * g;

    // 4-bit: scales of the 4 columns of each fragment that the lane's sums belong to; zero points of the row whose codes it holds.
    [[maybe_unused]] ScaleAt at[RN];
    [[maybe_unused]] uint32_t zero_at[RN];
    [[maybe_unused]] int groups = 1;
    if constexpr (kInt4) {
#pragma unroll
        for (int j = 0; j < RN; ++j) {
            const bool up = kGated && j % 2;
            const int total = up ? 2 * p.N : p.N;
            const int n = (up ? p.N : 0) + n0 + row_of(j);
            at[j] = scale_at(n + 4 * g, total);
            if constexpr (kZeros) zero_at[j] = static_cast<uint32_t>(n + r16 < total ? n + r16 : total - 1);
        }
        groups = (p.K + p.group - 1) / p.group;
    }

    constexpr int kWeights = kInt4 ? 1 : 4;   // 16-byte loads of a fragment's step
    constexpr int kScales = kInt4 ? kGroups : 1;
    struct Fetch {
        u32x4 w[RN][kWeights];
        u32x2 scale[kInt4 ? RN : 1][kScales];
        uint32_t zero[kZeros ? RN : 1][kScales];
    };
    const auto fetch = [&](Fetch& f, int turn) {
        const int step = first + turn * WK + part;
        if (step >= end) return;
        const int k0 = step * kStep;
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int s = 0; s < kWeights; ++s) {
                uint32_t off = w_off + static_cast<uint32_t>(row_of(j)) * static_cast<uint32_t>(pitch);
                if constexpr (kInt4) {
                    // Past K x is zero, and any code will do. The step's place counts for the buffer's end too: a row's last 16 bytes
                    // may reach past it.
                    f.w[j][0] = buf_load16(w_rsrc[kGated ? j % 2 : 0], off + static_cast<uint32_t>(k0 / 2));
                } else {
                    if (k0 + kStep > k_end && k0 + 32 * s + 8 * g >= k_end) off = kOob;
                    f.w[j][s] = buf_load16(w_rsrc[kGated ? j % 2 : 0], off, static_cast<uint32_t>(k0) * 2 + 64u * s);
                }
            }
        if constexpr (kInt4) {
#pragma unroll
            for (int c = 0; c < kScales; ++c) {
                const int group = step * kScales + c < groups ? step * kScales + c : groups - 1;
#pragma unroll
                for (int j = 0; j < RN; ++j) {
                    f.scale[j][c] = load_any<u32x2>(p.scale + group * p.ld_scale + at[j].from);
                    if constexpr (kZeros) f.zero[j][c] = (p.zero + group * p.ld_zero)[zero_at[j]];
                }
            }
        }
    };

    f32x4 acc[RM][RN];
    const f32x4 none{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = none;
    [[maybe_unused]] Decode<kBf16> decode;
    decode.init();
    const auto use = [&](const Fetch& f, int turn) {
        if (first + turn * WK + part >= end) return;
        if constexpr (kInt4) {
            constexpr int kPer = 4 / kGroups;   // MFMAs of a group
            u32x4 w[RN];
#pragma unroll
            for (int j = 0; j < RN; ++j) w[j] = kRun ? f.w[j][0] : transpose_rows(f.w[j][0]);
#pragma unroll
            for (int c = 0; c < kGroups; ++c) {
                half8 x[RM][kPer];
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int s = 0; s < kPer; ++s) x[i][s] = __builtin_bit_cast(half8, read_rows(turn, c * kPer + s, i));
                f32x4 t[RM][RN];
#pragma unroll
                for (int j = 0; j < RN; ++j) {
                    if constexpr (kZeros) decode.set_zero(f.zero[j][c]);
#pragma unroll
                    for (int s = 0; s < kPer; ++s) {
                        const half8 code = decode.template values<kZeros>(w[j][c * kPer + s]);
#pragma unroll
                        for (int i = 0; i < RM; ++i) t[i][j] = mfma16<kBf16>(code, x[i][s], s > 0 ? t[i][j] : none);
                    }
                }
#pragma unroll
                for (int j = 0; j < RN; ++j) {
                    const f32x4 scale = scales4<kBf16>(f.scale[j][c], at[j].shift);
#pragma unroll
                    for (int i = 0; i < RM; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(t[i][j][e], scale[e], acc[i][j][e]);
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                half8 x[RM];
#pragma unroll
                for (int i = 0; i < RM; ++i) x[i] = __builtin_bit_cast(half8, read_rows(turn, s, i));
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int j = 0; j < RN; ++j) acc[i][j] = mfma16<kBf16>(__builtin_bit_cast(half8, f.w[j][s]), x[i], acc[i][j]);
            }
        }
    };

    Fetch f[2];
    load_rows(0);
    fetch(f[0], 0);
    write_rows(0);
    load_rows(1);
    fetch(f[1], 1);
    for (int turn = 0; turn < turns; turn += 2) {
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            // This turn's rows are in LDS, and the other buffer's are read, for every wave past the barrier.
            if (turn + d < turns) {
                __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
                barrier_only();
                use(f[d], turn + d);
                write_rows(turn + d + 1);
                load_rows(turn + d + 2);
                fetch(f[d], turn + d + 2);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __syncthreads();
    auto* const join = reinterpret_cast<f32x4*>(lds);   // [waves][RM * RN][64]
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) join[(wave * RM * RN + i * RN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    constexpr int kPair = kGated ? 2 : 1;
    constexpr int kUnits = RM * RN / kPair;   // of a part of the columns: fragments, or gates with their ups
    for (int unit = wave; unit < kUnits * WN; unit += T::kWaves) {
        const int wn = unit / kUnits;
        const int f0 = unit % kUnits * kPair;
        f32x4 sum[1][kPair];
#pragma unroll
        for (int q = 0; q < kPair; ++q) {
            sum[0][q] = join[(wn * RM * RN + f0 + q) * 64 + lane];
#pragma unroll
            for (int w = 1; w < WK; ++w) sum[0][q] += join[((w * WN + wn) * RM * RN + f0 + q) * 64 + lane];
        }
        if (p.splits > 1 && !join_splits<kUnits * WN>(p, sum, static_cast<int>(blockIdx.x), split, unit, lane)) continue;
        store_sums<kForm, kBf16>(p, f0 / RN * 16 + r16, static_cast<int>(blockIdx.x) * (kWaveCols * WN) + wn * kWaveCols + row_of(f0 % RN) + 4 * g,
                                 sum[0][0], sum[0][kPair - 1], kInt4 ? Decode<kBf16>::kUnit : 1.0f);
    }
}

}  // namespace feather
