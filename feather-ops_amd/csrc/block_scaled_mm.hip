// The block-scaled fp8 product's host side and its streaming kernel (include/feather_block_ops.h, block_mm_common.h).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "block_mm_common.h"
#include "block_mm_tile.h"

namespace feather {
namespace {

constexpr int kStreamWaves = 8;

// Streaming kernel: a workgroup owns 16 RM x 16 RN outputs and its 8 waves take every eighth block of K each, reading both
// operands from memory straight into registers; their fp32 sums meet in LDS, added in wave order.
template <bool kAE5M2, bool kBE5M2, bool kByRow, int RM, int RN>
__global__ __launch_bounds__(kStreamWaves * 64) void block_stream_kernel(const BlockMmParams p) {
    __shared__ f32x4 join[kStreamWaves][RM * RN][64];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int tiles_n = (p.N + 16 * RN - 1) / (16 * RN);
    const int m0 = static_cast<int>(blockIdx.x) / tiles_n * 16 * RM;
    const int n0 = static_cast<int>(blockIdx.x) % tiles_n * 16 * RN;
    const int r16 = lane % 16;
    const int g = lane / 16;
    const rsrc_t a_rsrc = rows_rsrc(p.a, p.lda, m0, p.M, 16 * RM, p.K);
    const rsrc_t b_rsrc = rows_rsrc(p.b, p.ldb, n0, p.N, 16 * RN, p.K);
    const int blocks = (p.K + kBlock - 1) / kBlock;

    f32x4 acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int kb = wave; kb < blocks; kb += kStreamWaves) {
        i32x8 fa[RM], fb[RN];
        const auto fetch = [&](rsrc_t r, int row, int64_t ld) {
            u32x4 half[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = kb * kBlock + h * 64 + g * 16;
                half[h] = buf_load16(r, at < p.K ? static_cast<uint32_t>(row) * static_cast<uint32_t>(ld) + at : kOob);
                if (p.K % 16 != 0) half[h] = keep_bytes(half[h], p.K - at);
            }
            return join16(half[0], half[1]);
        };
        float sa[RM];
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            fa[i] = fetch(a_rsrc, 16 * i + r16, p.lda);
            const int m = m0 + 16 * i + r16;
            sa[i] = m < p.M ? p.a_scale[m * p.as_row + kb * p.as_block] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < RN; ++j) {
            fb[j] = fetch(b_rsrc, 16 * j + r16, p.ldb);
            const int n = n0 + 16 * j;
            if constexpr (kByRow) {
                f32x4 sb;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int col = n + 4 * g + e;
                    sb[e] = col < p.N ? p.b_scale[col * p.bs_row + kb * p.bs_block] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < RM; ++i) add_scaled(acc[i][j], mfma_block<kAE5M2, kBE5M2>(fb[j], fa[i]), sa[i] * sb);
            } else {
                const float sb = n < p.N ? p.b_scale[n / kBlock * p.bs_row + kb * p.bs_block] : 0.0f;
#pragma unroll
                for (int i = 0; i < RM; ++i) add_scaled(acc[i][j], mfma_block<kAE5M2, kBE5M2>(fb[j], fa[i]), sa[i] * sb);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) join[wave][i * RN + j][lane] = acc[i][j];
    __syncthreads();
    for (int f = wave; f < RM * RN; f += kStreamWaves) {
        f32x4 sum = join[0][f][lane];
#pragma unroll
        for (int w = 1; w < kStreamWaves; ++w) sum += join[w][f][lane];
        store_out(p, m0 + f / RN * 16 + r16, n0 + f % RN * 16 + 4 * g, sum);
    }
}

template <int RM, int RN>
void launch_stream(const BlockMmParams& p, bool a_e5m2, bool b_e5m2, bool by_row, hipStream_t stream) {
    const auto grid = static_cast<uint32_t>((p.M + 16 * RM - 1) / (16 * RM)) *
                      static_cast<uint32_t>((p.N + 16 * RN - 1) / (16 * RN));
    const auto go = [&](auto ae, auto be) {
        if (by_row) block_stream_kernel<ae(), be(), true, RM, RN><<<grid, kStreamWaves * 64, 0, stream>>>(p);
        else block_stream_kernel<ae(), be(), false, RM, RN><<<grid, kStreamWaves * 64, 0, stream>>>(p);
    };
    if (a_e5m2 && b_e5m2) go(std::true_type{}, std::true_type{});
    else if (a_e5m2) go(std::true_type{}, std::false_type{});
    else if (b_e5m2) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
}

template <typename T>
void launch_tile(const BlockMmParams& p, bool a_e5m2, bool b_e5m2, bool by_row, hipStream_t stream) {
    const auto grid = static_cast<uint32_t>((p.M + T::BM - 1) / T::BM) * static_cast<uint32_t>((p.N + T::BN - 1) / T::BN);
    const auto go = [&](auto ae, auto be) {
        if (by_row) block_tile_kernel<T, ae(), be(), true><<<grid, T::kThreads, 0, stream>>>(p);
        else block_tile_kernel<T, ae(), be(), false><<<grid, T::kThreads, 0, stream>>>(p);
    };
    if (a_e5m2 && b_e5m2) go(std::true_type{}, std::true_type{});
    else if (a_e5m2) go(std::true_type{}, std::false_type{});
    else if (b_e5m2) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
}

// 256 rows of a tile stay within 31-bit offsets, of codes and of scales.
constexpr int64_t kMaxLd = int64_t{4} << 20;
constexpr int64_t kMaxScaleStride = int64_t{1} << 20;

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
    return M >= 1 && M <= kMaxSize / 4 && N >= 1 && N <= kMaxSize / 4 && K >= 0 && K <= kMaxLd &&
           ((M + 15) / 16) * ((N + 15) / 16) <= kMaxSize;
}

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" int64_t feather_block_scaled_mm_workspace_bytes(int64_t M, int64_t N, int64_t K, bool) {
    return sizes_ok(M, N, K) ? 0 : -1;
}

extern "C" bool feather_block_scaled_mm(const uint8_t* a, int64_t lda, bool a_e5m2, const float* a_scale,
                                        int64_t a_scale_row, int64_t a_scale_block, const uint8_t* b, int64_t ldb,
                                        bool b_e5m2, const float* b_scale, int64_t b_scale_row, int64_t b_scale_block,
                                        bool b_by_row, const void* bias, void* c, int64_t ldc, int out_type, int64_t M,
                                        int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                                        hipStream_t stream) {
    if (!sizes_ok(M, N, K) || !type_ok(out_type)) return false;
    const int64_t need = feather_block_scaled_mm_workspace_bytes(M, N, K, b_by_row);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0))
        return false;
    if (K > 0 && (!a || !b || !a_scale || !b_scale || !on_16(a) || !on_16(b) || lda < K || ldb < K || lda % 16 != 0 ||
                  ldb % 16 != 0 || lda > kMaxLd || ldb > kMaxLd || a_scale_row < 0 || a_scale_row > kMaxScaleStride ||
                  b_scale_row < 0 || b_scale_row > kMaxScaleStride || a_scale_block < 0 || b_scale_block < 0 || !aligned_to_type(a_scale, FEATHER_FP32) ||
                  !aligned_to_type(b_scale, FEATHER_FP32)))
        return false;
    if (!c || ldc < N || ldc > kMaxSize || !aligned_to_type(c, out_type) || (bias && !aligned_to_type(bias, out_type)))
        return false;
    const int bytes = type_bytes(out_type);
    const bool store4 = (reinterpret_cast<uintptr_t>(c) & (4 * bytes - 1)) == 0 && ldc % 4 == 0;
    const bool store8 = rows_on_16(c, ldc, out_type) && N % 8 == 0 && on_16(bias);
    const BlockMmParams p{a, b, a_scale, b_scale, lda, ldb, a_scale_row, a_scale_block, b_scale_row, b_scale_block,
                          static_cast<int32_t>(M), static_cast<int32_t>(N), static_cast<int32_t>(K), 1, bias, c, ldc,
                          out_type, store4, store8, nullptr, nullptr};
    if (M <= 16) launch_stream<1, 1>(p, a_e5m2, b_e5m2, b_by_row, stream);
    else if (M <= 32) launch_stream<2, 1>(p, a_e5m2, b_e5m2, b_by_row, stream);
    else if (M <= 64) launch_stream<4, 2>(p, a_e5m2, b_e5m2, b_by_row, stream);
    else if (M <= 512) launch_tile<BlockTile<128, 128, 2, 2, 2>>(p, a_e5m2, b_e5m2, b_by_row, stream);
    else launch_tile<BlockTile<256, 256, 2, 4, 2>>(p, a_e5m2, b_e5m2, b_by_row, stream);
    return true;
}
