/*
 * C ABI of a decoder's feed-forward operators (libfeather_ops_gfx950.so): the gated block in 16 bits with its gradients, and
 * products with 4-bit weights that have one scale for each group of columns. Plain pointers and sizes, no torch types. No
 * counterpart in the reference.
 *
 * Types: FEATHER_BF16 and FEATHER_FP16 (feather_block_ops.h) for activations, 16-bit weights, scales and outputs alike.
 *
 * Every function enqueues on `stream` and returns true, or returns false and enqueues nothing where its contract is not met;
 * launch errors are left to the caller (hipGetLastError). No function allocates, synchronizes or keeps anything between calls.
 * Results are deterministic. Strides are in elements (of codes: bytes). Operands of products have rows on 16-byte boundaries
 * (strides are multiples of 8, at most 2^21) and, where a comment says padded, rows that can be read up to the next multiple of 8
 * values; outputs may have any alignment. Sizes: M < 2^29, N (rows of a weight) < 2^28, K at most 2^21, and few enough outputs for
 * a launch to have under 2^32 threads.
 *
 * Workspaces: the function's ..._workspace_bytes (0: none), 256-byte aligned. Its first 64 KiB are all zero before its first use
 * and left zero by every call; calls that share one must be ordered.
 */
#ifndef FEATHER_LINEAR_OPS_H
#define FEATHER_LINEAR_OPS_H

#include <stdbool.h>
#include <stdint.h>

#include "feather_block_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { FEATHER_SILU = 0, FEATHER_GELU = 1, FEATHER_GELU_TANH = 2 };

/*
 * y = act(x Wg^T + bg) * (x Wu^T + bu): sums, activation and product in fp32, rounded once.
 *   x       [M, K], K % 8 == 0
 *   weight  [2 F, K]: Wg's rows, then Wu's
 *   bias    2 F values, or null
 *   y       [M, F]
 *   kept    null, or for the backward fp32 [M, 2 F8] with F8 = F rounded up to 8: both sums with their bias, the gate's first,
 *           each in F8 columns; ld_kept >= 2 F8 and a multiple of 4, 16-byte aligned, under 2^22
 */
bool feather_gated_linear(const void* x, int64_t ldx, const void* weight, int64_t ld_weight, const void* bias, int type,
                          int activation, void* y, int64_t ldy, float* kept, int64_t ld_kept, int64_t M, int64_t F, int64_t K,
                          void* workspace, int64_t workspace_bytes, hipStream_t stream);
int64_t feather_gated_linear_workspace_bytes(int64_t M, int64_t F, int64_t K);

/*
 * The gradients of the two sums from y's: grad[m] = (dy up act'(gate), dy act(gate)), both rounded to `type`, [M, 2 F] with
 * stride ld_grad (>= 2 F8, a multiple of 8; columns from 2 F to 2 F8 are set to zero). sums: null, or fp32
 * [feather_gated_backward_parts(M, F), 2 F], contiguous: the column sums of groups of rows (of the unrounded values), for
 * feather_sum_rows (the bias's gradient).
 */
bool feather_gated_backward(const void* grad_y, int64_t ld_grad_y, const float* kept, int64_t ld_kept, int type, int activation,
                            void* grad, int64_t ld_grad, float* sums, int64_t M, int64_t F, hipStream_t stream);
int64_t feather_gated_backward_parts(int64_t M, int64_t F);

/*
 * c[m, n] = sum over k of a(m, k) b(n, k) + bias[n] (N values, or null), in fp32, rounded once to `type`.
 *   a  [M, K], or [K, M] where a_across;  b  [N, K], or [K, N] where b_across (a_across needs b_across). Stored across, an
 *      operand's rows are padded; stored along, they are padded with zeros.
 */
bool feather_product(const void* a, int64_t lda, bool a_across, const void* b, int64_t ldb, bool b_across, const void* bias,
                     int type, void* c, int64_t ldc, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                     hipStream_t stream);
int64_t feather_product_workspace_bytes(int64_t M, int64_t N, int64_t K);

/*
 * 4-bit weights [N, K]: value (n, k) is (q - z) * s with the code q (0 .. 15) and, of its group of `group` (32, 64 or 128)
 * columns, the scale s and the zero point z (0 .. 15).
 *   codes  two to a byte, the even column in the low half; rows of (K + 1) / 2 bytes, ld_codes apart, a multiple of 4 up to 2^22;
 *          4-byte aligned; rows can be read up to a multiple of 4 bytes
 *   scale  of `type`, group by group: (n, g) at g * ld_scale + n, with 4 values to a group at least
 *   zero   one byte each, the same with ld_zero; or null: 8
 */

/*
 * y = x W^T + bias (gated false), or act(x Wg^T + bg) * (x Wu^T + bu) with W's first N rows the gates' and N more the ups'
 * (gated true: W, scale, zero and bias have 2 N rows), rounded once. x [M, K], padded to K % 8 == 0 with zeros. Up to 64 rows
 * codes are taken as they are, each group's sum times its scale in fp32. Of more rows each is computed so or, most of them, with the
 * weight rounded to `type` first; which ones depends on the sizes alone. For more than 64 rows 15 times a scale is within the type's
 * range, and the codes' rows start on 16-byte boundaries.
 */
bool feather_int4_linear(const void* x, int64_t ldx, const uint8_t* codes, int64_t ld_codes, const void* scale,
                         int64_t ld_scale, const uint8_t* zero, int64_t ld_zero, int group, const void* bias, int type, bool gated,
                         int activation, void* y, int64_t ldy, int64_t M, int64_t N, int64_t K, void* workspace,
                         int64_t workspace_bytes, hipStream_t stream);
int64_t feather_int4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gated);

/* Whether feather_int4_linear takes M rows of these codes and is at least as fast as feather_int4_dequantize and a product in 16
 * bits, where every row has the rounded weight. True up to 64 rows. */
bool feather_int4_linear_direct(const uint8_t* codes, int64_t ld_codes, int64_t M, int64_t N, int64_t K, bool gated);

/* w [N, K] of `type` from 4-bit weights, each value rounded once; ldw a multiple of 8, columns from K to the next multiple of 8
 * are set to zero. */
bool feather_int4_dequantize(const uint8_t* codes, int64_t ld_codes, const void* scale, int64_t ld_scale, const uint8_t* zero,
                             int64_t ld_zero, int group, int type, void* w, int64_t ldw, int64_t N, int64_t K, hipStream_t stream);

/*
 * 4-bit weights of w [N, K] (row stride ldw). Without zero points (zero null) a group's scale is its largest magnitude / 7; with
 * them its range, extended to zero, / 15, and z the code of zero. Scales are rounded to `type` first, and codes are the nearest to
 * w / s + z. A group whose scale is zero has codes z. A group with a NaN or an infinity has a scale of NaN or infinity, and every
 * value that is computed from it is NaN.
 */
bool feather_int4_quantize(const void* w, int64_t ldw, int type, int group, uint8_t* codes, int64_t ld_codes, void* scale,
                           int64_t ld_scale, uint8_t* zero, int64_t ld_zero, int64_t N, int64_t K, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FEATHER_LINEAR_OPS_H */
