// The streaming kernel of the block-scaled fp8 product, for few rows: both operands go from memory straight into registers,
// and a workgroup's waves split K. What bounds it is the reading of b: one row against 14336 x 4096 takes 14.2 us, against
// 4096 x 14336 12.4, where reading the same rows in the same order and nothing else took 11.1-11.8, and in one linear run
// 9.6-10.1. With more rows a's come from L2 once for each workgroup, which is why RN grows with them: 24 rows 16.2 and 16.6.
#pragma once

#include "block_mm_common.h"

namespace feather {

// RM x RN 16 x 16 output fragments per workgroup, kWaves waves that take every kWaves-th block of K each, with kDepth blocks
// in flight per wave.
template <int RM_, int RN_, int kWaves_, int kDepth_>
struct BlockStream {
    static constexpr int RM = RM_, RN = RN_, kWaves = kWaves_, kDepth = kDepth_;
    static constexpr int kThreads = 64 * kWaves;
    static_assert(RN <= 8 && 8 % RN == 0, "a workgroup's columns have one square scale");
};

template <typename T, bool kAE5M2, bool kBE5M2, bool kByRow>
__global__ __launch_bounds__(T::kThreads) void block_stream_kernel(const BlockMmParams p) {
    constexpr int RM = T::RM, RN = T::RN;
    __shared__ f32x4 join[T::kWaves][RM * RN][64];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int m0 = static_cast<int>(blockIdx.y) * 16 * RM;
    const int n0 = static_cast<int>(blockIdx.x) * 16 * RN;
    const int r16 = lane % 16;
    const int g = lane / 16;
    const rsrc_t a_rsrc = rows_rsrc(p.a, p.lda, m0, p.M, 16 * RM, p.K);
    const rsrc_t b_rsrc = rows_rsrc(p.b, p.ldb, n0, p.N, 16 * RN, p.K);
    const int all_blocks = (p.K + kBlock - 1) / kBlock;
    const int split = static_cast<int>(blockIdx.z);
    const int first = p.splits > 1 ? split * all_blocks / p.splits : 0;
    const int blocks = p.splits > 1 ? (split + 1) * all_blocks / p.splits : all_blocks;   // this workgroup's end
    const uint32_t a_off = static_cast<uint32_t>(r16) * static_cast<uint32_t>(p.lda) + 16 * g;
    const uint32_t b_off = static_cast<uint32_t>(r16) * static_cast<uint32_t>(p.ldb) + 16 * g;
    // Scales, as buffers of this workgroup's rows: strides within 2^20 and 64 rows stay in 31 bits, blocks are walked by
    // moving the base.
    uint32_t sa_off[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int row = 16 * i + r16;
        sa_off[i] = m0 + row < p.M ? static_cast<uint32_t>(row * p.as_row) * 4u : kOob;
    }
    const float* const sa_base = p.a_scale + m0 * p.as_row;
    constexpr int kScalesB = kByRow ? RN : 1;
    uint32_t sb_off[kScalesB][4];
    if constexpr (kByRow) {
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 16 * j + 4 * g + e;
                sb_off[j][e] = n0 + col < p.N ? static_cast<uint32_t>(col * p.bs_row) * 4u : kOob;
            }
    }
    const float* const sb_base = p.b_scale + (kByRow ? static_cast<int64_t>(n0) : n0 / kBlock) * p.bs_row;

    struct Fetch {
        u32x4 a[RM][2], b[RN][2];
        float sa[RM], sb[kScalesB][kByRow ? 4 : 1];
    };
    // Block kb, the operand that comes from memory first; one scale for all columns comes through the scalar cache.
    const auto fetch = [&](Fetch& f, int kb) {
        const uint32_t base = static_cast<uint32_t>(kb) * kBlock;
        const bool there[2] = {static_cast<int>(base) + 16 * g < p.K, static_cast<int>(base) + 64 + 16 * g < p.K};
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                f.b[j][h] = buf_load16(
                    b_rsrc, there[h] ? b_off + 16u * j * static_cast<uint32_t>(p.ldb) + base + 64 * h : kOob);
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                f.a[i][h] = buf_load16(a_rsrc, there[h] ? a_off + 16u * i * static_cast<uint32_t>(p.lda) + base + 64 * h : kOob);
        const auto load4 = [](const float* from, uint32_t off) {
            return __builtin_bit_cast(
                float, __builtin_amdgcn_raw_buffer_load_b32(make_rsrc(from, 0x7fffffffu), static_cast<int>(off), 0, 0));
        };
#pragma unroll
        for (int i = 0; i < RM; ++i) f.sa[i] = load4(sa_base + kb * p.as_block, sa_off[i]);
        if constexpr (kByRow) {
#pragma unroll
            for (int j = 0; j < RN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) f.sb[j][e] = load4(sb_base + kb * p.bs_block, sb_off[j][e]);
        } else {
            f.sb[0][0] = sb_base[kb * p.bs_block];
        }
    };

    f32x4 acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const auto use = [&](Fetch& f, int kb) {
        if (p.K % 16 != 0 && kb == all_blocks - 1) {   // the last block ends inside a 16-byte piece
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int valid = p.K - kb * kBlock - 64 * h - 16 * g;
#pragma unroll
                for (int j = 0; j < RN; ++j) f.b[j][h] = keep_bytes(f.b[j][h], valid);
#pragma unroll
                for (int i = 0; i < RM; ++i) f.a[i][h] = keep_bytes(f.a[i][h], valid);
            }
        }
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const f32x4 t = mfma_block<kAE5M2, kBE5M2>(join16(f.b[j][0], f.b[j][1]), join16(f.a[i][0], f.a[i][1]));
                if constexpr (kByRow) {
                    add_scaled(acc[i][j], t, f.sa[i] * f32x4{f.sb[j][0], f.sb[j][1], f.sb[j][2], f.sb[j][3]});
                } else {
                    add_scaled(acc[i][j], t, f.sa[i] * f.sb[0][0]);
                }
            }
    };

    Fetch f[T::kDepth];
#pragma unroll
    for (int d = 0; d < T::kDepth; ++d)
        if (first + wave + d * T::kWaves < blocks) fetch(f[d], first + wave + d * T::kWaves);
    for (int kb = first + wave; kb < blocks; kb += T::kDepth * T::kWaves) {
#pragma unroll
        for (int d = 0; d < T::kDepth; ++d) {
            if (kb + d * T::kWaves < blocks) use(f[d], kb + d * T::kWaves);
            if (kb + (d + T::kDepth) * T::kWaves < blocks) fetch(f[d], kb + (d + T::kDepth) * T::kWaves);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) join[wave][i * RN + j][lane] = acc[i][j];
    __syncthreads();
    for (int f = wave; f < RM * RN; f += T::kWaves) {
        f32x4 sum[1][1] = {{join[0][f][lane]}};
#pragma unroll
        for (int w = 1; w < T::kWaves; ++w) sum[0][0] += join[w][f][lane];
        if (p.splits > 1) {
            const int tile = static_cast<int>(blockIdx.y * gridDim.x + blockIdx.x);
            if (!join_splits<RM * RN>(p, sum, tile, split, f, lane)) continue;
        }
        store_out(p, m0 + f / RN * 16 + r16, n0 + f % RN * 16 + 4 * g, sum[0][0]);
    }
}

}  // namespace feather
