// The tile kernel of the products with 4-bit weights, for more rows than few: linear_tile.h's, with the weight's stages in LDS as
// codes. Each wave takes them to 16 bits in registers, (q - z) s rounded once, between its matrix instructions. So that no value
// is taken twice in a workgroup its 4 waves lie side by side, each with all of the tile's rows and 64 of its 256 columns: 128 KB
// of LDS reads a stage either way, of 256 rows.
//
// The rounding of the weights adds to the output's: together they are off by 2.14e-3 of the norm in bf16 and 2.75e-4 in fp16, where
// the output's alone is 1.66e-3 and 2.07e-4. (Codes as they are would want fp32 sums of each group beside the 256 that a lane holds.)
//
// What bounds it are instructions: a stage of 256 rows has 128 MFMAs and some 500 others of a wave, which issues one in four
// clocks. A stage takes 1.4 us on one CU (linear_tile.h's 1.0), and 1000 x 4096 -> 14336 100-115 us, where dequantizing takes 37
// and the product 86. From about 2000 rows on the other way is faster (4096 x 4096 -> 14336 411 us, 366).
#pragma once

#include <utility>

#include "int4_common.h"
#include "linear_tile.h"

namespace feather {

// f(0) .. f(n - 1), the numbers constants. (Loops as long as these, of as much, the compiler doesn't unroll.)
template <typename F, int... kI>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, kI...>) {
    (f(std::integral_constant<int, kI>{}), ...);
}

template <int n, typename F>
__device__ __forceinline__ void each(F&& f) {
    each(static_cast<F&&>(f), std::make_integer_sequence<int, n>{});
}

template <int BM_>
struct Int4Tile {
    static constexpr int BM = BM_, BN = 256;            // 256 or 128 rows
    static constexpr int kPerCu = 256 / BM;             // workgroups of a CU
    static constexpr int kWaves = 4;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int RM = BM / 16;                  // fragments of a wave
    static constexpr int RN = BN / 16 / kWaves;
    static constexpr int kAUnit = BM * 128;             // bytes of an operand's stage
    static constexpr int kBUnit = BN * 32;
    static constexpr int kStages = 3 * kAUnit + 2 * kBUnit;   // as linear_tile.h's
    template <bool kGated>
    using Out = OutStage<RM, kGated ? RN / 2 : RN>;
    template <bool kGated>
    static constexpr int kLdsBytes = kStages > kWaves * Out<kGated>::kBytes ? kStages : kWaves * Out<kGated>::kBytes;
    static constexpr int kALoads = BM / 32;             // of a wave and stage
    static constexpr int kBLoads = BN / 32 / kWaves;
    static constexpr int kMfmas = RM * RN;              // of half a stage
    static constexpr int kBarrier = kMfmas / 8;         // the MFMA of the second half before which the workgroup meets
    static constexpr int kDecode = kMfmas / 4;          // the MFMA of the second half from which codes are there
};

// A wave's scales and zero points: a lane holds those of column 16 (lane / 16) + lane % 16 of its 64, as one word. What a
// fragment's lanes need of it is that row of 16 lanes in all four.
__device__ __forceinline__ void spread_rows(uint32_t v, uint32_t (&out)[4]) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(a[0], a[0], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[1], a[1], false, false);
    out[0] = b[0];
    out[1] = b[1];
    out[2] = c[0];
    out[3] = c[1];
}

// 8 codes of a column to 16 bits in steps of about an instruction that go between the MFMAs. bf16: q s - z s in fp32, exact,
// rounded as it is packed; a code's byte, read as a float of 8 bits (e4m3), is q / 512, and two at a time are converted and multiplied
// by 512. fp16: codes in the mantissas of 1024 + q and 1024 + 16 q, from where a multiplication and addition takes them to q - z,
// exactly.
template <bool kBf16>
struct Decoder {
    static constexpr int kSetup = 4;
    static constexpr int kSteps = kSetup + 16;
    uint32_t even, odd;        // bf16: the codes, in bytes
    float scale, offset;
    float lo[2], hi[2];        // two pairs
    uint32_t scales, offsets;  // fp16: twice each, 1024 + z and 64 + z
    uint32_t pair, one;

    __device__ __forceinline__ void init() {
        one = 0x64006400u;
        asm volatile("" : "+v"(one));   // in a register, for one instruction with the mask
    }
    template <int kStep>
    __device__ __forceinline__ void step(uint32_t code, uint32_t word, u32x4& out) {
        if constexpr (kBf16) {
            constexpr bool kTop = kStep >= kSetup + 8;
            constexpr int e = (kStep - kSetup) % 8;
            if constexpr (kStep == 0) {
                even = code & 0x0f0f0f0fu;
            } else if constexpr (kStep == 1) {
                odd = code >> 4 & 0x0f0f0f0fu;
            } else if constexpr (kStep == 2) {
                offset = static_cast<float>(word >> 16 & 255u);
                scale = __builtin_bit_cast(float, word << 16);
            } else if constexpr (kStep == 3) {
                offset *= -scale;
            } else if constexpr (e < 2) {
                const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(e == 0 ? even : odd, 512.0f, kTop);
                (e == 0 ? lo : hi)[0] = v[0];
                (e == 0 ? lo : hi)[1] = v[1];
            } else if constexpr (e < 4) {
                lo[e - 2] = __builtin_fmaf(lo[e - 2], scale, offset);
            } else if constexpr (e < 6) {
                hi[e - 4] = __builtin_fmaf(hi[e - 4], scale, offset);
            } else {
                out[(kTop ? 2 : 0) + e - 6] = pack2<FEATHER_BF16>(lo[e - 6], hi[e - 6]);
            }
        } else {
            constexpr int q = (kStep - kSetup) / 4, k = (kStep - kSetup) % 4;
            if constexpr (kStep == 0) {
                scales = __builtin_amdgcn_perm(0u, word, perm_sel(0, 1, 0, 1));
            } else if constexpr (kStep == 1) {
                offsets = word >> 16;
            } else if constexpr (kStep == 2) {
                offsets |= offsets << 20;
            } else if constexpr (kStep == 3) {
                offsets |= 0x54006400u;
            } else if constexpr (k == 0) {
                pair = __builtin_amdgcn_perm(0u, code, perm_sel(q, kZeroByte, q, kZeroByte));
            } else if constexpr (k == 1) {
                pair = (pair & 0x00f0000fu) | one;
            } else if constexpr (k == 2) {
                const half2v part{static_cast<_Float16>(1.0f), static_cast<_Float16>(0.0625f)};
                pair = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, pair), part,
                                                                              -__builtin_bit_cast(half2v, offsets)));
            } else {
                out[q] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, pair) * __builtin_bit_cast(half2v, scales));
            }
        }
    }
};

template <typename T, Form kForm, bool kBf16>
__global__ __launch_bounds__(T::kThreads) __attribute__((amdgpu_waves_per_eu(T::kPerCu, T::kPerCu)))
void int4_tile_kernel(const Int4Params p) {
    constexpr int RM = T::RM, RN = T::RN;
    static_assert(RN == 4, "a fragment for each 16 lanes");
    constexpr bool kGated = kForm != Form::kPlain;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::template kLdsBytes<kGated>];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    constexpr int kCols = kGated ? T::BN / 2 : T::BN;   // outputs of a tile's row
    const int tiles = p.tiles_m * p.tiles_n;
    const int split = p.splits > 1 ? static_cast<int>(blockIdx.x) / tiles : 0;
    const int tile = static_cast<int>(blockIdx.x) - split * tiles;
    int tm, tn;
    tile_of_block(tile, tiles, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = p.m_first + tm * T::BM;
    const int col0 = p.n_first + tn * kCols + wave * (kCols / T::kWaves);   // the wave's first output
    const int all = (p.K + 63) / 64;
    const int first = static_cast<int>(static_cast<int64_t>(split) * all / p.splits);
    const int last = static_cast<int>(static_cast<int64_t>(split + 1) * all / p.splits) - 1;   // loaded first, as linear_tile.h's
    const int stages = last + 1 - first;
    const int r16 = lane % 16, g = lane / 16;

    Operand<T::BM, false, false> a;
    a.init(p.a, p.lda, m0, p.M, p.K, wave, lane, 0);

    // The wave's codes: two loads of 32 columns (gated: of gates, then of ups), 32 bytes each.
    rsrc_t code_rsrc[2];
    const int bytes = ((p.K + 1) / 2 + 3) & ~3;   // that can be read of a row
#pragma unroll
    for (int d = 0; d < 2; ++d) {
        const int n = col0 + (kGated ? 0 : 32 * d);
        const int rows = p.N - n < 32 ? p.N - n : 32;
        code_rsrc[d] = make_rsrc(p.codes + (n + (kGated && d ? static_cast<int64_t>(p.N) : 0)) * p.ld_codes,
                                 rows > 0 ? static_cast<uint32_t>(rows - 1) * static_cast<uint32_t>(p.ld_codes) + bytes : 0u);
    }
    const uint32_t code_off = static_cast<uint32_t>(lane / 2) * static_cast<uint32_t>(p.ld_codes) + lane % 2 * 16u;
    const auto load_b = [&](int d, int stage, bool live, uint32_t unit) {
        dma16(code_rsrc[d], lds + unit + (2 * wave + d) * 1024, live ? code_off + static_cast<uint32_t>(stage) * 32u : kOob);
    };
    // A fragment's column in LDS.
    const auto column = [&](int j) { return 64 * wave + (kGated ? j % 2 * 32 + j / 2 * 16 : 16 * j) + r16; };

    // The lane's column of scales and zero points. Without zero points loads give 0, which becomes 8.
    const int own = kGated ? col0 + g / 2 * 16 + r16 : col0 + lane;
    const int own_row = own + (kGated && g % 2 ? p.N : 0);
    const uint32_t scale_off = own < p.N ? static_cast<uint32_t>(own_row) * 2u : kOob;
    const uint32_t zero_off = own < p.N ? static_cast<uint32_t>(own_row) : kOob;
    const uint32_t weight_rows = kGated ? 2 * p.N : p.N;
    const uint32_t no_zero = p.zero ? 0u : 8u;
    const uint32_t zero_bytes = p.zero ? weight_rows : 0u;
    const int group_shift = p.group == 32 ? 5 : p.group == 64 ? 6 : 7;
    uint32_t raw_scale[2], raw_zero[2];
    const auto group_row = [&](const auto* rows, int64_t ld, int s, int stage, uint32_t bytes) {
        const int k = stage * 64 + 32 * s;
        const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(k) >> group_shift) * static_cast<uint32_t>(ld);
        return make_rsrc(rows + at, k < p.K ? bytes : 0u);
    };
    const auto load_scale = [&](int s, int stage) {
        raw_scale[s] = __builtin_amdgcn_raw_buffer_load_b16(group_row(p.scale, p.ld_scale, s, stage, weight_rows * 2u),
                                                            static_cast<int>(scale_off), 0, 0);
    };
    const auto load_zero = [&](int s, int stage) {
        raw_zero[s] = __builtin_amdgcn_raw_buffer_load_b8(group_row(p.zero, p.ld_zero, s, stage, zero_bytes), static_cast<int>(zero_off), 0, 0);
    };

    f32x4 acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 x[RM], w[2][RN];   // w: of both halves of a stage
    uint32_t code[2][RN], word[2][RN];
    using D = Decoder<kBf16>;
    D decoder;
    decoder.init();

    const auto make_words = [&](int s) { spread_rows(raw_scale[s] | (raw_zero[s] ^ no_zero) << 16, word[s]); };
    const auto read_code = [&](int s, int j, uint32_t unit) {
        code[s][j] = *reinterpret_cast<const uint32_t*>(lds + unit + column(j) * 32 + s * 16 + g * 4);
    };
    // Step e of a half's 4 columns.
    const auto decode_step = [&](int s, auto e) {
        constexpr int j = e / D::kSteps;
        decoder.template step<e % D::kSteps>(code[s][j], word[s][j], w[s][j]);
    };

    uint32_t ua = 0, na = T::kAUnit, fa = 2 * T::kAUnit, ub = 3 * T::kAUnit, nb = ub + T::kBUnit;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        load_scale(s, last);
        load_zero(s, last);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int d = 0; d < T::kALoads; ++d) a.load(d, t ? first : last, t < stages, lds + (t ? na : ua), wave);
#pragma unroll
        for (int d = 0; d < T::kBLoads; ++d) load_b(d, t ? first : last, t < stages, t ? nb : ub);
    }
    a.start(first + 1);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::kALoads + T::kBLoads));
    barrier_only();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        make_words(s);
#pragma unroll
        for (int j = 0; j < RN; ++j) read_code(s, j, ub);
        load_scale(s, first);
        load_zero(s, first);
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) x[i] = a.read(lds, ua, i, 0);
    each<RN * D::kSteps>([&](auto e) { decode_step(0, e); });

    const auto multiply = [&](int m, int s) {
        const int i = m / RN;
        const int j = i % 2 ? RN - 1 - m % RN : m % RN;
        acc[i][j] = mfma16<kBf16>(__builtin_bit_cast(half8, w[s][j]), __builtin_bit_cast(half8, x[i]), acc[i][j]);
    };
    // The steps of a half's decoding, spread evenly over its MFMAs from kFrom on: those of MFMA m.
    const auto decode_at = [&](auto m, auto from, int s) {
        constexpr int kSteps = RN * D::kSteps, kFrom = from, kSlots = T::kMfmas - kFrom;
        if constexpr (m >= kFrom) {
            constexpr int kAt = (m - kFrom) * kSteps / kSlots, kNext = (m - kFrom + 1) * kSteps / kSlots;
            each<kNext - kAt>([&](auto e) { decode_step(s, std::integral_constant<int, kAt + e>{}); });
        }
    };
    for (int t = 0; t < stages; ++t) {
        // First half: row i's fragment is used and then that of the second half is read in its place; the second half's codes
        // become values, a's loads of stage t + 2 are issued.
        each<T::kMfmas>([&](auto m) {
            multiply(m, 0);
            if constexpr (m % RN == RN - 1) x[m / RN] = a.read(lds, ua, m / RN, 1);
            static_assert(T::kMfmas == 8 * T::kALoads, "a's loads fill the half");
            if constexpr (m % 8 == 1) a.load_next(m / 8, t + 2 < stages, lds, fa, wave);
            decode_at(m, std::integral_constant<int, 0>{}, 1);
            __builtin_amdgcn_sched_barrier(0);
        });
        // Second half: past the barrier stage t is read and stage t + 1 has landed, for every wave.
        each<T::kMfmas>([&](auto m) {
            if constexpr (m == T::kBarrier) {
                __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::kALoads));
                barrier_only();
            }
            multiply(m, 1);
            if constexpr (m >= T::kBarrier) {
                constexpr int n = m - T::kBarrier;
                if constexpr (n == 0 || n == 2) each<2>([&](auto j) { read_code(0, n + j, nb); });
                if constexpr (n == 4 || n == 6) each<2>([&](auto j) { read_code(1, n - 4 + j, nb); });
                if constexpr (n == 1) each<T::kBarrier / RN>([&](auto i) { x[i] = a.read(lds, na, i, 0); });
                if constexpr (n == 4 || n == 8) make_words((n - 4) / 4);
                if constexpr (n == 10 || n == 18) load_scale((n - 10) / 8, first + t + 1);
                if constexpr (n == 14 || n == 22) load_zero((n - 14) / 8, first + t + 1);
                if constexpr (m % RN == RN - 1) x[m / RN] = a.read(lds, na, m / RN, 0);
                if constexpr (n % 8 == 5 && n / 8 < T::kBLoads) load_b(n / 8, first + t + 1, t + 2 < stages, ub);
                decode_at(m, std::integral_constant<int, T::kDecode>{}, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        a.advance();
        const uint32_t freed = ua;
        ua = na;
        na = fa;
        fa = freed;
        const uint32_t other = ub;
        ub = nb;
        nb = other;
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) asm volatile("" : "+a"(acc[i][j]));   // as linear_tile.h's
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // the last loads write LDS
    __builtin_amdgcn_s_waitcnt(kLgkm0Imm);
    barrier_only();
    if (p.splits > 1 && !join_splits<T::kWaves>(p, acc, tile, split, wave, lane)) return;
    finish<kForm, kBf16>(p, acc, m0, col0, lane, lds + wave * T::template Out<kGated>::kBytes);
}

}  // namespace feather
