/*
 * C ABI of microscaled 4-bit floating point (MI355X / gfx950): the quantiser, products of two quantised operands, products of a few 16-bit rows
 * with quantised weights, and a layer of experts for a few tokens.  Same library (libdlblas_fp8_gemm.so), same conventions as
 * include/dlblas_decoder.h: nothing is allocated, synchronised or kept, every launch is a kernel on `stream`, 0 = enqueued, negative DLB_ERR_* =
 * rejected with a reason in dlb_last_error() and nothing enqueued.
 *
 * The format (OCP microscaling, version 1.0): 32 consecutive columns of a row share a scale 2^(s - 127), one byte s, 255 = NaN; an element is e2m1, a
 * sign above three bits that stand for 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Codes lie two a byte, the even column in the low half; scales beside them:
 * [rows, K / 2] and [rows, K / 32], contiguous.
 */
#ifndef DLBLAS_MXFP4_H_
#define DLBLAS_MXFP4_H_

#include "dlblas_fp8_gemm.h"
#include "dlblas_fp8_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* widest row of an operand */
#define DLB_MXFP4_MAX_COLUMNS (1 << 22)

/*
 * Codes and scales of rows: s = max(floor(log2 max |x|) - 2, -127) + 127 per group, q = x 2^(127 - s) to nearest, ties to the even code, magnitudes
 * above 6 to 6, signs kept.  A group that holds an infinity or a NaN has s = 255 and codes 0.
 *
 *   x [rows, K] bf16 / fp16 / fp32 (dtype, DLB_IN_*), row stride x_row_stride, aligned to its elements;  q [rows, K/2], 4-byte aligned;  s [rows, K/32]
 */
int dlb_mxfp4_quant(const void* x, int64_t x_row_stride, int dtype, void* q, void* s, int64_t rows, int64_t K, void* stream);

/* Bytes of scratch dlb_mxfp4_gemm needs. */
size_t dlb_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K);

/*
 * c[m, n] = sum over the groups g of 2^(a_s[m, g] + b_s[n, g] - 254) sum_{k in g} a[m, k] b[n, k]; fp32 sums in an order that depends on the sizes
 * alone, one rounding at the end.
 *
 *   a [M, K/2], b [N, K/2]      codes, 16-byte aligned;  a_s [M, K/32], b_s [N, K/32]  scales, 4-byte aligned
 *   c [M, N]                    bf16 / fp16 / fp32 (out_dtype, DLB_IN_*), contiguous
 *   workspace                   16-byte aligned, dlb_mxfp4_gemm_workspace_bytes(M, N, K), no initialisation; calls that can overlap need their own
 *
 * K % 32 == 0, at most DLB_MXFP4_MAX_COLUMNS.
 */
int dlb_mxfp4_gemm(const void* a, const void* b, const void* a_s, const void* b_s, void* c, int64_t M, int64_t N, int64_t K, int out_dtype,
                   void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DLBLAS_MXFP4_H_ */
