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

/*
 * y[m, n] = sum over the groups g of 2^(s[n, g] - 127) sum_{k in g} x[m, k] q[n, k]; fp32 sums, one rounding at the end.  Meant for up to a few dozen rows: the weights are read once per 16 of them,
 * beside each other.
 *
 *   x [M, K]     bf16 / fp16 (dtype), row stride x_row_stride (even, at most 2^23), 4-byte aligned
 *   q [N, K/2]   codes, 16-byte aligned;  s [N, K/32] scales
 *   y [M, N]     dtype, contiguous
 *
 * K % 32 == 0, at most DLB_MXFP4_MAX_COLUMNS.
 */
int dlb_mxfp4_weight_gemm(const void* x, int64_t x_row_stride, int dtype, const void* q, const void* s, void* y, int64_t M, int64_t N, int64_t K,
                          void* stream);

/* what dlb_few_token_experts takes at most */
#define DLB_FEW_TOKENS 64
#define DLB_FEW_TOPK 16
#define DLB_FEW_EXPERTS 1024
#define DLB_FEW_NUMBERS (1 << 29) /* tokens * topk * I */
/* weight types of dlb_few_token_experts: e4m3fn with fp32 scales of 128 x 128, or the 4-bit format above */
#define DLB_WEIGHTS_E4M3 0
#define DLB_WEIGHTS_MXFP4 1

/* Bytes of scratch dlb_few_token_experts needs. */
size_t dlb_few_token_experts_workspace_bytes(int64_t tokens, int64_t topk, int64_t I);

/*
 * A layer of experts for a few tokens:
 *   out[t] = sum over the slots j with 0 <= ids[t, j] < experts of weights[t, j] Down[e] (silu(Gate[e] x[t]) * (Up[e] x[t])),  e = ids[t, j]
 * Products, sums and what lies between the products in fp32, the result rounded once.  Zeros for a token
 * without an expert here; slots that name one expert twice count both weights.  The order of all sums depends on the routing and the sizes alone.
 * What lies between the products meets Down exactly down to 2^-126.
 *
 *   x       [tokens, H]     bf16 / fp16 (dtype), row stride x_row_stride (even, at most 2^23), 4-byte aligned
 *   ids     [tokens, topk]  int32 / int64 (ids_dtype, DLB_IDX_*) through two strides;  weights [tokens, topk] fp32, contiguous
 *   up_q    [experts, 2 I, H], rows of Gate, then rows of Up;  down_q [experts, H, I]: e4m3fn, or codes of half that width, 16-byte aligned
 *   up_s, down_s            scales: [experts, ceil(rows / 128), columns / 128] fp32, or [experts, rows, columns / 32] bytes
 *   out     [tokens, H]     dtype, contiguous
 *   workspace               4-byte aligned, dlb_few_token_experts_workspace_bytes(tokens, topk, I), no initialisation; calls that can overlap need
 *                           their own
 *
 * tokens at most 64, topk 16, experts 1024; H and I multiples of 128 with e4m3 weights, of 32 with 4-bit ones, at most 2^20.
 */
int dlb_few_token_experts(const void* x, int64_t x_row_stride, int dtype, const void* ids, int ids_dtype, int64_t ids_stride_m, int64_t ids_stride_k,
                          const float* weights, int weight_type, const void* up_q, const void* up_s, const void* down_q, const void* down_s, void* out,
                          int64_t tokens, int64_t topk, int64_t experts, int64_t H, int64_t I, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DLBLAS_MXFP4_H_ */
