// The streaming kernels for few rows: weights (16-bit or 4-bit) and activations go from memory straight into registers, and a
// workgroup's waves split K. What bounds them is the reading of the weight.
#pragma once

#include "int4_common.h"

namespace feather {

// RM x RN 16 x 16 output fragments per workgroup (gated: RN / 2 of gates, as many of ups), kWaves waves that take every
// kWaves-th step of 128 k's, with kDepth steps in flight.
template <int RM_, int RN_, int kWaves_, int kDepth_>
struct LinearStream {
    static constexpr int RM = RM_, RN = RN_, kWaves = kWaves_, kDepth = kDepth_;
    static constexpr int kThreads = 64 * kWaves;
};

constexpr int kStep = 128;

// Four outputs of row m at columns n .. n + 3.
template <bool kBf16>
__device__ __forceinline__ void store4(const LinearParams& p, int m, int n, f32x4 v) {
    if (m >= p.M || n >= p.N) return;
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

// A row's sums to outputs: gate and up of columns n .. n + 3, or (plain) the sums themselves.
template <Form kForm, bool kBf16>
__device__ __forceinline__ void store_sums(const LinearParams& p, int m, int n, f32x4 sum, f32x4 up) {
    if (m >= p.M || n >= p.N) return;
    sum += bias4<kBf16>(p.bias, n, p.N);
    if constexpr (kForm != Form::kPlain) {
        up += bias4<kBf16>(p.bias, int64_t{p.N} + n, int64_t{2} * p.N);
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
__global__ __launch_bounds__(T::kThreads) void linear_stream_kernel(const std::conditional_t<kGroups != 0, Int4Params, LinearParams> p) {
    constexpr bool kInt4 = kGroups != 0;
    constexpr int RM = T::RM, RN = T::RN;
    constexpr bool kGated = kForm != Form::kPlain;
    static_assert(!kGated || RN % 2 == 0, "gates and ups go in pairs");
    constexpr int kCols = 16 * (kGated ? RN / 2 : RN);
    __shared__ f32x4 join[T::kWaves][RM * RN][64];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int n0 = static_cast<int>(blockIdx.x) * kCols;
    const int split = static_cast<int>(blockIdx.y);
    const int r16 = lane % 16;
    const int g = lane / 16;
    const int all = (p.K + kStep - 1) / kStep;
    const int first = static_cast<int>(static_cast<int64_t>(split) * all / p.splits) + wave;
    const int end = static_cast<int>(static_cast<int64_t>(split + 1) * all / p.splits);

    // Weights: fragment j is 16 rows from row_of(j).
    const auto row_of = [&](int j) { return kGated ? 16 * (j / 2) : 16 * j; };
    const int here = p.N - n0 < kCols ? p.N - n0 : kCols;
    const bool edge = here < kCols;
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
    const uint32_t records = static_cast<uint32_t>(here - 1) * static_cast<uint32_t>(pitch) + static_cast<uint32_t>(row_bytes);
    const rsrc_t w_rsrc[2] = {make_rsrc(weight + n0 * pitch, records),
                              make_rsrc(weight + (kGated ? p.N + static_cast<int64_t>(n0) : n0) * pitch, records)};
    // A lane's k's of a step: 8 of each MFMA, 32 s + 8 g; of 4-bit groups of 128, which one lane may hold any part of, 32 g + 8 s, as
    // its 16 bytes of codes have them (other groups' dwords change lanes first).
    constexpr bool kRun = kGroups == 1;
    const uint32_t w_off = static_cast<uint32_t>(r16) * static_cast<uint32_t>(pitch) + 16u * g;
    const rsrc_t x_rsrc = make_rsrc(p.a, static_cast<uint32_t>(p.M - 1) * static_cast<uint32_t>(p.lda * 2) + static_cast<uint32_t>((p.K + 7) & ~7) * 2u);
    uint32_t x_off[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i)
        x_off[i] = 16 * i + r16 < p.M ? static_cast<uint32_t>(16 * i + r16) * static_cast<uint32_t>(p.lda * 2) + (kRun ? 64u : 16u) * g : kOob;
    const auto k_of = [&](int s) { return kRun ? 32 * g + 8 * s : 32 * s + 8 * g; };
    constexpr uint32_t kNext = kRun ? 16 : 64;   // bytes of x from one MFMA's to the next one's

    // 4-bit: scales and zero points of the lane's 4 columns of each fragment.
    [[maybe_unused]] ScaleAt at[RN];
    [[maybe_unused]] int groups = 1;
    if constexpr (kInt4) {
#pragma unroll
        for (int j = 0; j < RN; ++j)
            at[j] = kGated && j % 2 ? scale_at(p.N + n0 + row_of(j) + 4 * g, 2 * p.N) : scale_at(n0 + row_of(j) + 4 * g, p.N);
        groups = (p.K + p.group - 1) / p.group;
    }

    constexpr int kWeights = kInt4 ? 1 : 4;   // 16-byte loads of a fragment's step
    constexpr int kScales = kInt4 ? kGroups : 1;
    struct Fetch {
        u32x4 w[RN][kWeights];
        u32x2 scale[kInt4 ? RN : 1][kScales];
        uint32_t zero[kZeros ? RN : 1][kScales];
    };
    const auto fetch = [&](Fetch& f, int step) {
        const uint32_t k0 = static_cast<uint32_t>(step) * kStep;
        const bool whole = step * kStep + kStep <= p.K;
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int s = 0; s < kWeights; ++s) {
                uint32_t off = w_off + static_cast<uint32_t>(row_of(j)) * static_cast<uint32_t>(pitch);
                if constexpr (kInt4) {
                    // the step's place counts for the buffer's end too: a row's last 16 bytes may reach past it
                    f.w[j][0] = buf_load16(w_rsrc[kGated ? j % 2 : 0], off + k0 / 2);
                } else {
                    if (!whole && step * kStep + 32 * s + 8 * g >= p.K) off = kOob;
                    f.w[j][s] = buf_load16(w_rsrc[kGated ? j % 2 : 0], off, k0 * 2 + 64u * s);
                }
            }
        if constexpr (kInt4) {
#pragma unroll
            for (int c = 0; c < kScales; ++c) {
                const int group = step * kScales + c < groups ? step * kScales + c : groups - 1;
#pragma unroll
                for (int j = 0; j < RN; ++j) {
                    f.scale[j][c] = load_any<u32x2>(p.scale + group * p.ld_scale + at[j].from);
                    if constexpr (kZeros) f.zero[j][c] = load_any<uint32_t>(p.zero + group * p.ld_zero + at[j].from);
                }
            }
        }
    };
    struct Rows {
        u32x4 x[RM][4];
    };
    const auto fetch_rows = [&](Rows& f, int step) {
        const uint32_t k0 = static_cast<uint32_t>(step) * kStep;
        const bool whole = step * kStep + kStep <= p.K;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                uint32_t off = x_off[i];
                if (!whole && step * kStep + k_of(s) >= p.K) off = kOob;
                f.x[i][s] = buf_load16(x_rsrc, off, k0 * 2 + kNext * s);
            }
    };

    f32x4 acc[RM][RN];
    const f32x4 none{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = none;
    [[maybe_unused]] const uint32_t one = code_one<kBf16>();
    const auto use = [&](const Fetch& f, const Rows& rows) {
        if constexpr (kInt4) {
            constexpr int kPer = 4 / kGroups;       // MFMAs of a group
            u32x4 w[RN];
#pragma unroll
            for (int j = 0; j < RN; ++j) w[j] = kRun ? f.w[j][0] : transpose_rows(f.w[j][0]);
#pragma unroll
            for (int c = 0; c < kGroups; ++c) {
                half8 x[RM][kPer];
                // What the codes' offsets take: of fixed ones the sums start there, of zero points it is the sum of x.
                constexpr bool kSums = kZeros || kBf16;
                f32x4 sums[RM];
#pragma unroll
                for (int i = 0; i < RM; ++i) {
                    sums[i] = none;
#pragma unroll
                    for (int s = 0; s < kPer; ++s) {
                        x[i][s] = order8(rows.x[i][c * kPer + s]);
                        if constexpr (kSums) sums[i] = mfma16<kBf16>(constant8<kBf16, !kZeros>(), x[i][s], sums[i]);
                    }
                }
                f32x4 t[RM][RN];
#pragma unroll
                for (int s = 0; s < kPer; ++s)
#pragma unroll
                    for (int j = 0; j < RN; ++j) {
                        const half8 code = decode8<kBf16>(w[j][c * kPer + s], one);
#pragma unroll
                        for (int i = 0; i < RM; ++i)
                            t[i][j] = mfma16<kBf16>(code, x[i][s], s > 0 ? t[i][j] : kSums && !kZeros ? sums[i] : none);
                    }
#pragma unroll
                for (int j = 0; j < RN; ++j) {
                    const f32x4 scale = scales4<kBf16>(f.scale[j][c], edge, at[j].shift);
                    f32x4 off = none;
                    if constexpr (kZeros) {
                        off = zeros4(f.zero[j][c], edge, at[j].shift);
#pragma unroll
                        for (int e = 0; e < 4; ++e) off[e] = kCodeBias<kBf16> - off[e];
                    }
#pragma unroll
                    for (int i = 0; i < RM; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = t[i][j][e];
                            if constexpr (kZeros) v = __builtin_fmaf(off[e], sums[i][e], v);
                            acc[i][j][e] = __builtin_fmaf(v, scale[e], acc[i][j][e]);
                        }
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int j = 0; j < RN; ++j)
                        acc[i][j] = mfma16<kBf16>(__builtin_bit_cast(half8, f.w[j][s]), __builtin_bit_cast(half8, rows.x[i][s]), acc[i][j]);
        }
    };

    // Weights kDepth steps ahead; activations, which come from cache, one.
    Fetch f[T::kDepth];
    constexpr int kSets = RM > 2 ? 1 : 2;
    Rows rows[kSets];
#pragma unroll
    for (int d = 0; d < T::kDepth; ++d) {
        if (first + d * T::kWaves < end) fetch(f[d], first + d * T::kWaves);
        if (d == 0 && kSets > 1 && first < end) fetch_rows(rows[0], first);
    }
    static_assert(T::kDepth % kSets == 0, "rows go through two sets of registers");
    for (int step = first; step < end; step += T::kDepth * T::kWaves) {
#pragma unroll
        for (int d = 0; d < T::kDepth; ++d) {
            const int at_step = step + d * T::kWaves;
            const int ahead = kSets > 1 ? at_step + T::kWaves : at_step;
            if (ahead < end) fetch_rows(rows[(d + 1) % kSets], ahead);
            if (at_step < end) use(f[d], rows[d % kSets]);
            if (at_step + T::kDepth * T::kWaves < end) fetch(f[d], at_step + T::kDepth * T::kWaves);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) join[wave][i * RN + j][lane] = acc[i][j];
    __syncthreads();
    constexpr int kPair = kGated ? 2 : 1;
    for (int f0 = kPair * wave; f0 < RM * RN; f0 += kPair * T::kWaves) {
        f32x4 sum[1][kPair];
#pragma unroll
        for (int q = 0; q < kPair; ++q) {
            sum[0][q] = join[0][f0 + q][lane];
#pragma unroll
            for (int w = 1; w < T::kWaves; ++w) sum[0][q] += join[w][f0 + q][lane];
        }
        if (p.splits > 1 && !join_splits<RM * RN / kPair>(p, sum, static_cast<int>(blockIdx.x), split, f0 / kPair, lane)) continue;
        store_sums<kForm, kBf16>(p, f0 / RN * 16 + r16, n0 + row_of(f0 % RN) + 4 * g, sum[0][0], sum[0][kPair - 1]);
    }
}

}  // namespace feather
