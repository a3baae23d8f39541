/*
 * C ABI of the steps around the products of a decoder block (MI355X / gfx950): RMS norm with the residual's addition and the
 * 1 x 128 quantiser, tokens sorted by expert and back with their gradients, products of a few rows with 4-bit weights.
 * Same library (libdlblas_fp8_gemm.so), same conventions as include/dlblas_fp8_gemm.h: device pointers and sizes only, nothing is
 * allocated or synchronised, work is enqueued on `stream`, 0 = enqueued, negative DLB_ERR_* = rejected with a reason in
 * dlb_last_error() and nothing enqueued.  Every launch is a kernel, so all of them can be captured into a HIP graph.  No call keeps
 * anything; scratch is an argument of the calls that need it, and calls that can overlap in time need their own.
 *
 * Element types: DLB_IN_BF16 / DLB_IN_F16 / DLB_IN_F32 (include/dlblas_fp8_gemm.h).  Row strides are in elements; the last dimension
 * is contiguous; any element-aligned address will do unless said otherwise.  Outputs must not overlap inputs.
 */
#ifndef DLBLAS_DECODER_H_
#define DLBLAS_DECODER_H_

#include "dlblas_fp8_gemm.h"
#include "dlblas_fp8_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* widest row of the norms and of dlb_moe_unpermute_backward */
#define DLB_NORM_MAX_COLUMNS 32768
/* experts of dlb_moe_permute */
#define DLB_SORT_MAX_EXPERTS 1024
/* element type of dlb_moe_permute beside DLB_IN_*: e4m3fn with fp32 scales of 1 x 128 */
#define DLB_ROWS_E4M3 3

/*
 * h = x + residual rounded to the element type (h = x without a residual), y = h * w / sqrt(mean(h^2) + eps); fp32 inside, one
 * rounding at the store.  The sum of squares is fp32 as well: rows whose sum passes 2^128 (|h| about 10^17 throughout) give y = 0, or
 * NaN where they hold an infinity.
 *
 *   x, residual, y, sum  [rows, H]  one element type (dtype); residual NULL: none, and sum is not written
 *   weight               [H]        the same type, or fp32 (weight_dtype)
 */
int dlb_rms_norm(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, int dtype,
                 const void* weight, int weight_dtype, void* y, int64_t y_row_stride, void* sum, int64_t sum_row_stride,
                 int64_t rows, int64_t H, float eps, void* stream);

/*
 * The same with y quantised per 128 columns instead of stored: s = max(max |y|, quant_eps) / 448, q = e4m3(y / s).  y is not
 * rounded to the element type in between.  A group that holds an infinity or a NaN dequantises to NaN.
 *
 *   q  [rows, H]      e4m3fn, contiguous, 8-byte aligned; H % 128 == 0
 *   s  [rows, H/128]  fp32, element (m, g) at s[m * s_stride_m + g * s_stride_k]
 */
int dlb_rms_norm_quant(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, int dtype,
                       const void* weight, int weight_dtype, void* q, float* s, int64_t s_stride_m, int64_t s_stride_k,
                       void* sum, int64_t sum_row_stride, int64_t rows, int64_t H, float eps, float quant_eps, void* stream);

/* Bytes of scratch dlb_rms_norm_backward needs for dw (none otherwise). */
size_t dlb_rms_norm_backward_workspace_bytes(int64_t rows, int64_t H);

/*
 * The gradients of dlb_rms_norm from its h:  dx = r (w dy - h r^2 / H sum(w dy h)) + dsum,  dw = sum over the rows of dy h r.
 * dx is the gradient of x and of the residual alike.  The order of all sums is fixed.
 *
 *   dy, dsum, h, dx  [rows, H]  dtype; dsum (gradient of sum) may be NULL
 *   dw               [H]        weight_dtype, or NULL: not wanted
 *   workspace        4-byte aligned, dlb_rms_norm_backward_workspace_bytes(rows, H), no initialisation
 */
int dlb_rms_norm_backward(const void* dy, int64_t dy_row_stride, const void* dsum, int64_t dsum_row_stride, const void* h,
                          int64_t h_row_stride, int dtype, const void* weight, int weight_dtype, void* dx, int64_t dx_row_stride,
                          void* dw, int64_t rows, int64_t H, float eps, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of scratch dlb_moe_permute needs. */
size_t dlb_moe_permute_workspace_bytes(int64_t tokens, int64_t topk, int64_t experts);

/*
 * Tokens copied next to the other tokens of each expert they are routed to, and the tables that say where.  Slots (t, j) with
 * 0 <= ids[t, j] < experts are ordered by (expert, t, j); expert e gets the rows from row_start[e] on, its count rounded up to
 * `alignment`.  Slots whose row would be num_rows or more get none.  rows[r] = x[source[r] / topk], zeros where source[r] < 0.
 *
 *   ids        [tokens, topk]  int32 / int64 (ids_dtype, DLB_IDX_*) through two strides; topk <= 64
 *   x          [tokens, H]     bf16 / fp16 / fp32 (DLB_IN_*) or e4m3fn (DLB_ROWS_E4M3: H % 128 == 0, rows of x and `rows` 16-byte
 *                              aligned)
 *   x_s        [tokens, H/128] fp32 through two strides with e4m3fn rows, else NULL
 *   row_index  [tokens, topk]  int32, contiguous, OUT: row of every slot, -1 where it has none
 *   source     [num_rows]      int32, OUT: slot t * topk + j of every row, -1 where it holds none
 *   m_indices  [num_rows]      int32, OUT: expert of every row of a span, -1 past the last span (the form that
 *                              dlb_fp8_gemm_grouped_contiguous takes with alignment 128)
 *   row_start, row_end [experts] int32, OUT: rows of every expert that hold a slot (the form dlb_fp8_gemm_grouped_ragged and
 *                              dlb_w4_gemm take); at most num_rows
 *   rows       [num_rows, H]   contiguous, OUT;   rows_s [num_rows, H/128] fp32, contiguous, OUT with e4m3fn rows
 *
 * With H = 0 the tables alone are written.
 */
int dlb_moe_permute(const void* ids, int ids_dtype, int64_t ids_stride_m, int64_t ids_stride_k, const void* x, int64_t x_row_stride,
                    int dtype, const float* x_s, int64_t xs_stride_m, int64_t xs_stride_k, int32_t* row_index, int32_t* source,
                    int32_t* m_indices, int32_t* row_start, int32_t* row_end, void* rows, float* rows_s, int64_t tokens, int64_t H,
                    int64_t topk, int64_t experts, int64_t alignment, int64_t num_rows, void* workspace, size_t workspace_bytes,
                    void* stream);

/*
 * out[t] = sum over the slots j with 0 <= row_index[t, j] < num_rows, in slot order, of weights[t, j] * rows[row_index[t, j]]; an fp32
 * FMA chain, one rounding at the end; zeros for a token without a row.  Also the gradient of dlb_moe_permute (weights NULL).
 *
 *   rows [num_rows, H], out [tokens, H]  dtype;  weights [tokens, topk] fp32, contiguous, or NULL: all one
 */
int dlb_moe_unpermute(const void* rows, int64_t rows_row_stride, int dtype, const int32_t* row_index, const float* weights, void* out,
                      int64_t out_row_stride, int64_t tokens, int64_t H, int64_t topk, int64_t num_rows, void* stream);

/*
 * The gradients of dlb_moe_unpermute with the tables of dlb_moe_permute (every row is named by one slot at most):
 * drows[row] = weights[t, j] * dout[t], zeros in rows without a slot; dweights[t, j] = sum over the columns of rows[row] * dout[t], 0 for
 * a slot without a row.
 *
 *   dweights [tokens, topk] fp32, contiguous, or NULL: not wanted (rows is not read then and may be NULL)
 */
int dlb_moe_unpermute_backward(const void* dout, int64_t dout_row_stride, const void* rows, int64_t rows_row_stride, int dtype,
                               const int32_t* row_index, const int32_t* source, const float* weights, void* drows,
                               int64_t drows_row_stride, float* dweights, int64_t tokens, int64_t H, int64_t topk, int64_t num_rows,
                               void* stream);

/* Bytes of scratch dlb_w4_gemm needs; experts = 0 for one matrix without row ranges (with them none is needed). */
size_t dlb_w4_gemm_workspace_bytes(int64_t rows, int64_t N, int64_t K, int64_t experts);

/*
 * y[m, n] = sum over the groups g of K of s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g]); fp32 sums, one rounding at the end.
 * The sums of a group are those of x (16 + q) and x (16 + z): they are off by up to 24 * 2^-24 of 62 sum |x|, as long as fp32 holds
 * 32 sum |x| (fp16 rows: always; bf16 rows: |x| below 8 * 10^34 will do).  Past that, and for an infinity, whose sign and weight the
 * definition would keep, the two sums leave NaN.
 *
 *   x    [rows, K]         bf16 / fp16 (dtype), row stride x_row_stride (even, at most 2^24), 4-byte aligned
 *   q    [experts, N, K/2] 4-bit codes, the even column in the low half of a byte; contiguous, 16-byte aligned
 *   s    [experts, N, K/group] scales, bf16 / fp16 (s_dtype), contiguous
 *   z    the same shape, one byte each (0 ... 16; a byte above makes its column of y NaN), or NULL: 8 everywhere
 *   y    [rows, N]         dtype, row stride y_row_stride
 *   row_start, row_end [experts] int32 on the device: expert e multiplies the rows [row_start[e], row_end[e]), clamped to
 *        [0, rows]; ranges share no row, rows of no expert are not written.  NULL with experts = 1: every row
 *   workspace              4-byte aligned, dlb_w4_gemm_workspace_bytes(rows, N, K, row_start ? experts : 0), no initialisation
 *
 * group 32, 64 or 128; K % group == 0; K at most 2^24.  Meant for up to a few dozen rows (per expert): the weights are read once per
 * 32 of them.
 */
int dlb_w4_gemm(const void* x, int64_t x_row_stride, int dtype, const void* q, const void* s, int s_dtype, const void* z, void* y,
                int64_t y_row_stride, const int32_t* row_start, const int32_t* row_end, int64_t rows, int64_t N, int64_t K,
                int64_t group, int64_t experts, void* workspace, size_t workspace_bytes, void* stream);

/*
 * 4-bit codes of a weight, per group of columns: without z  s = max |w| / 7, q = clamp(round(w / s) + 8, 0, 15);  with z
 * s = (max(w, 0) - min(w, 0)) / 15, z = round(-min(w, 0) / s), q = clamp(round(w / s) + z, 0, 15); s rounded to the type of w before it
 * divides.  A group of zeros has s = 0, and so has one whose s rounds to 0.  A group that holds an infinity or a NaN, or whose max - min
 * passes fp32, has s = NaN and dequantises to NaN.
 *
 *   w [rows, K] bf16 / fp16, row stride w_row_stride;  q [rows, K/2], 4-byte aligned;  s [rows, K/group] of w's type;  z or NULL
 */
int dlb_w4_quant(const void* w, int64_t w_row_stride, int dtype, void* q, void* s, void* z, int64_t rows, int64_t K, int64_t group,
                 void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DLBLAS_DECODER_H_ */
