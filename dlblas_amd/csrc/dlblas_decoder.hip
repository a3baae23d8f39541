// C ABI of the steps around the products of a decoder block: argument validation and launches.
// The declarations and the contract of every entry point are in include/dlblas_decoder.h.
#include "../../include/dlblas_decoder.h"

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "moe_sort.h"
#include "rms_norm.h"
#include "w4_gemm.h"

namespace dlb {
namespace {

int finish(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(DLB_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return DLB_OK;
}

bool bad_dtype(int d) { return d < kInBf16 || d > kInF32; }
int64_t size_of(int d) { return d == kInF32 ? 4 : 2; }
bool off_elements(const void* p, int dtype) { return misaligned(p, size_of(dtype)); }

// Calls f with the type as a constant.
template <typename F>
void with_type(int dtype, F f) {
  if (dtype == kInBf16)
    f(std::integral_constant<int, kInBf16>());
  else if (dtype == kInF16)
    f(std::integral_constant<int, kInF16>());
  else
    f(std::integral_constant<int, kInF32>());
}
template <typename F>
void with_flag(bool flag, F f) {
  flag ? f(std::true_type()) : f(std::false_type());
}
template <int... C, typename F>
void with_chunks(int chunks, F f) {
  (void)((chunks == C && (f(std::integral_constant<int, C>()), true)) || ...);
}

// ---- norms ------------------------------------------------------------------------------------------------------------

// Threads of a workgroup and chunks of eight columns per thread for rows of H.
struct RowShape {
  int threads, chunks;
};
RowShape row_shape(int64_t H, int want_chunks) {
  const int64_t chunks = ceil_div(H, 8);
  int c = want_chunks;
  while (c < 4 && ceil_div(chunks, c) > kNormMaxThreads) c *= 2;
  return {static_cast<int>(ceil_div(ceil_div(chunks, c), 64) * 64), c};
}

// Rows of a multiple of eight up to 256 columns share waves: 2^20 x 128, the norm 266 -> 98 us (5.5 TB/s), with quantiser 324 -> 105, its gradient
// 2807 -> 296; 64 x 128 3.9 -> 3.8.
constexpr int kNarrowThreads = 256;  // of a workgroup
constexpr std::integral_constant<int, 1> kOne;
constexpr std::integral_constant<int, 64> kWave;
template <typename F>
bool with_lanes(int64_t H, F f) {
  if (H > 256) return false;
  H <= 128 ? f(std::integral_constant<int, 16>()) : f(std::integral_constant<int, 32>());
  return true;
}

// A grid of `blocks` workgroups in two dimensions.
dim3 row_grid(int64_t blocks) {
  constexpr int64_t kMost = 1 << 21;  // of up to 1024 threads, of which one dimension holds fewer than 2^32
  return dim3(static_cast<unsigned>(std::min(blocks, kMost)), static_cast<unsigned>(ceil_div(blocks, kMost)));
}

int check_norm(const void* x, const void* residual, int dtype, const void* weight, int weight_dtype, const void* sum, int64_t rows,
               int64_t H) {
  if (bad_dtype(dtype)) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16 / F32", dtype);
  if (weight_dtype != dtype && weight_dtype != kInF32)
    return fail(DLB_ERR_BAD_DTYPE, "weight_dtype %d is neither the rows' type nor DLB_IN_F32", weight_dtype);
  if (rows < 0 || H < 0) return fail(DLB_ERR_BAD_SHAPE, "negative dimension (rows=%lld H=%lld)", (long long)rows, (long long)H);
  if (rows > (1ll << 31) - 1 || H > DLB_NORM_MAX_COLUMNS)
    return fail(DLB_ERR_BAD_SHAPE, "rows=%lld / H=%lld beyond the supported range (H at most %d)", (long long)rows, (long long)H,
                DLB_NORM_MAX_COLUMNS);
  if (rows == 0 || H == 0) return DLB_OK;
  if (!x || !weight || (residual && !sum)) return fail(DLB_ERR_NULL_POINTER, "x, weight, or sum of a call with a residual is NULL");
  if (off_elements(x, dtype) || off_elements(residual, dtype) || off_elements(sum, dtype) || off_elements(weight, weight_dtype))
    return fail(DLB_ERR_ALIGNMENT, "a tensor is not aligned to its elements");
  return DLB_OK;
}

template <bool QUANT>
int launch_norm(const NormArgs& a, int dtype, hipStream_t st) {
  const auto launch = [&](auto t, auto res, auto whole, auto c, auto lanes, int threads, int beside) {
    hipLaunchKernelGGL((rms_norm_kernel<t(), QUANT, res(), whole(), c(), lanes()>), row_grid(ceil_div(a.rows, beside)), dim3(threads, beside), 0, st, a);
  };
  with_type(dtype, [&](auto t) {
    with_flag(a.res != nullptr, [&](auto res) {
      if (a.H % 8 == 0) {
        constexpr std::true_type whole;
        if (with_lanes(a.H, [&](auto lanes) { launch(t, res, whole, kOne, lanes, lanes(), kNarrowThreads / lanes()); })) return;
      }
      const RowShape shape = row_shape(a.H, 2);  // 8192 x 7168 quantised: one chunk a thread 95 us, two 78, four 78; a single row 3.5, 3.7, 4.9
      with_chunks<1, 2, 4>(shape.chunks, [&](auto c) {
        if (QUANT || a.H % 8 == 0)
          launch(t, res, std::true_type(), c, kWave, shape.threads, 1);
        else if constexpr (!QUANT)
          launch(t, res, std::false_type(), c, kWave, shape.threads, 1);
      });
    });
  });
  return finish("rms_norm");
}

// Shares of dw that the backward pass leaves, one of a workgroup (4096 x 7168: 256 of them 65 us, 384 61, 512 51, 768 64, 1024 58).  Of fewer
// than eight waves more where each has eight rows or more, for waves enough: 131072 x 512 390 -> 113 us, 65536 x 2048
// 307 -> 197; of narrow rows one of a wave.
int norm_grad_shares(int64_t rows, int64_t H) {
  if (H % 8 != 0 || H > 256) {
    const int64_t most = std::max<int64_t>(512, 4096 / ceil_div(H, 512));
    return static_cast<int>(std::min(rows, std::max<int64_t>(512, std::min(most, rows / 8))));
  }
  const int64_t rows_each = kNarrowThreads / (H <= 128 ? 16 : 32);
  return static_cast<int>(std::min<int64_t>(ceil_div(rows, rows_each), 512) * (kNarrowThreads / 64));
}

// ---- tokens by expert -------------------------------------------------------------------------------------------------

int check_rows(int64_t tokens, int64_t H, int64_t topk, int64_t num_rows) {
  if (tokens < 0 || H < 0 || num_rows < 0)
    return fail(DLB_ERR_BAD_SHAPE, "negative dimension (tokens=%lld H=%lld num_rows=%lld)", (long long)tokens, (long long)H, (long long)num_rows);
  if (topk < 1 || topk > kSortMaxTopk) return fail(DLB_ERR_BAD_SHAPE, "topk=%lld is not 1 ... %d", (long long)topk, kSortMaxTopk);
  if (tokens * topk > (1ll << 31) - 1 || num_rows > (1ll << 31) - 1 || tokens > (1ll << 31) - 1)
    return fail(DLB_ERR_BAD_SHAPE, "tokens * topk=%lld or num_rows=%lld does not fit the int32 tables", (long long)(tokens * topk), (long long)num_rows);
  if (H > (1ll << 28)) return fail(DLB_ERR_BAD_SHAPE, "H=%lld beyond the supported range", (long long)H);
  return DLB_OK;
}

// Whether a launch of its own adds up the counts of the workgroups of slots before each, instead of each reading all of them: tables of 8192
// tokens x 8 slots, 256 experts 13.1 and 13.7 us, 16384 13.5 and 17.8, 60000 19.9 and 42.6, 10^6 190 and 7733; 32 experts 8192 11.2 and 8.9,
// 60000 16.5 and 13.5, 131072 26.6 and 28.1.
bool sort_scans(int64_t blocks, int64_t experts) { return blocks * experts > 16384; }
int64_t sort_blocks(int64_t slots) { return slots > 0 ? ceil_div(slots, kSortBlockSlots) : 1; }

// ---- 4-bit weights ----------------------------------------------------------------------------------------------------

// What a product runs as: K split over the waves of a workgroup, or neighbouring tiles sharing x, in K slices of `chunks` chunks.
struct W4Plan {
  bool shared;
  int mt, slices, chunks;
};
constexpr int kW4Cus = 256;

int w4_columns(int mt) { return mt == 1 ? 64 : 128; }                       // of a workgroup that shares x
int w4_chunk(int mt) { return mt == 1 ? 2 * kW4Unit : kW4Unit; }           // columns of x

// rows_each: of one matrix.  Above 16 rows tiles of 32 x 32 (32 x 7168 x 7168 20.3 -> 17.9 us, 32 experts x 16 rows x 7168 x 2048 87 -> 66);
// above 8 rows per expert too, because experts have more than the mean.  Below, whichever of the two kernels is estimated faster, in us:
//   shared x   a chunk of a workgroup alone on its CU is about one; rounds over the chip x chunks, which go in pairs.  Workgroups beside
//              each other on a CU overlap, the more the less they have to compute.  With slices a second launch and the sums' way through
//              memory at 5 TB/s.  Slices that this picks, and others, in one run: 1 x 7168 x 18432 nine 20.6, two 24.0, four 21.2; 16 rows nine 24.7, two
//              25.0, four 26.0; 1 x 7168 x 7168 four 11.6, one 16.1, seven 12.5; 64 x 36864 x 7168 two 87, one 92, seven 99.
//   K over the waves   a launch, the columns of K, each the longer the more rows there are, further rounds, at most 2.4 TB/s.
// Measured, K over the waves / shared: 1 x 512 x 2048 4.3 / 5.9, 16 x 512 x 2048 5.6 / 6.9, 1 x 2112 x 7168 7.6 / 7.6, 16 x 2112 x 7168 11.8 / 8.4,
// 1 x 128 x 18432 14.5 / 8.4, 16 x 1024 x 14336 21.3 / 10.2, 1 x 16384 x 1024 9.2 / 4.8, 1 x 4096 x 4096 5.8 / 6.9, 8 experts x 1 row x 512 x 7168
// 8.1 / 17.1, 32 experts x 4 rows x 4096 x 7168 197 / 102.
W4Plan w4_plan(int64_t rows_each, bool by_expert, int64_t matrices, int64_t N, int64_t K) {
  const int mt = rows_each <= (by_expert ? 8 : 16) ? 1 : 2;
  const W4Plan waves{false, 1, 1, 0};
  if (N * (K / 128) < 4) return waves;  // fewer scales than a lane of the other kernel reads at once
  const int chunks = static_cast<int>(ceil_div(K, w4_chunk(mt)));
  W4Plan best{true, mt, 1, chunks};
  const int64_t base = matrices * ceil_div(N, w4_columns(mt)) * ceil_div(rows_each, 16 * mt);
  const double beside = rows_each <= 4 ? 0.75 : 0.85, rows = static_cast<double>(rows_each), n = static_cast<double>(N), k = static_cast<double>(K);
  double best_cost = 1e30;
  for (int slices = 1; slices <= (by_expert ? 1 : 16) && slices <= chunks; ++slices) {
    const int each = static_cast<int>(ceil_div(chunks, slices));
    if (ceil_div(chunks, each) != slices) continue;
    const int64_t rounds = ceil_div(base * slices, kW4Cus);
    const double sums = slices > 1 ? 3 + 0.3 * slices + 8e-6 / 5 * slices * rows * n : 0;
    const double cost = (rounds == 1 ? 1 : beside * static_cast<double>(rounds)) * ((each + 1) / 2 * 2) + sums;
    if (cost < best_cost) best_cost = cost, best.slices = slices, best.chunks = each;
  }
  if (mt == 1) {
    const double rounds = static_cast<double>(ceil_div(matrices * ceil_div(N, 16), kW4Cus));
    const double by_columns = 6.2e-4 * k * (1 + 0.055 * rows) + 1.5 * (rounds - 1), by_bytes = static_cast<double>(matrices) * n * k / 2 / 2.4e6;
    if (2.9 + std::max(by_columns, by_bytes) < best_cost + (best.slices > 1 ? 0.5 : 2.6) + 0.05 * rows) return waves;
  }
  return best;
}

template <int T, int GROUPS, bool ZEROS>
void launch_w4(const W4Args& a, const W4Plan& plan, int64_t y_blocks, float* sums, hipStream_t st) {
  if (!plan.shared) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.N, 16)), static_cast<unsigned>(y_blocks));
    hipLaunchKernelGGL((w4_gemm_kernel<T, GROUPS, ZEROS>), grid, dim3(64 * kW4Waves), 0, st, a);
    return;
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(a.N, w4_columns(plan.mt))), static_cast<unsigned>(y_blocks), static_cast<unsigned>(plan.slices));
  const dim3 block(64 * kW4Waves);
  float* const to = plan.slices > 1 ? sums : nullptr;
  if (plan.mt == 2)
    hipLaunchKernelGGL((w4_gemm_shared_kernel<T, GROUPS, ZEROS, 2, 2, 1, 4>), grid, block, 0, st, a, to, plan.chunks);
  else if (!a.row_start && a.rows <= 4)
    hipLaunchKernelGGL((w4_gemm_shared_kernel<T, GROUPS, ZEROS, 1, 1, 2, 1>), grid, block, 0, st, a, to, plan.chunks);
  else
    hipLaunchKernelGGL((w4_gemm_shared_kernel<T, GROUPS, ZEROS, 1, 1, 2, 4>), grid, block, 0, st, a, to, plan.chunks);
  if (plan.slices > 1)
    hipLaunchKernelGGL(w4_sum_kernel<T>, dim3(static_cast<unsigned>(ceil_div(a.rows * a.N, 256))), dim3(256), 0, st, sums, a.y, a.y_rs, a.rows, a.N, plan.slices);
}

}  // namespace
}  // namespace dlb

extern "C" {

int dlb_rms_norm(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, int dtype,
                 const void* weight, int weight_dtype, void* y, int64_t y_row_stride, void* sum, int64_t sum_row_stride,
                 int64_t rows, int64_t H, float eps, void* stream) {
  using namespace dlb;
  clear_error();
  if (int rc = check_norm(x, residual, dtype, weight, weight_dtype, sum, rows, H)) return rc;
  if (rows == 0 || H == 0) return DLB_OK;
  if (!y) return fail(DLB_ERR_NULL_POINTER, "y is NULL");
  if (off_elements(y, dtype)) return fail(DLB_ERR_ALIGNMENT, "y is not aligned to its elements");
  if (y_row_stride < H || (residual && sum_row_stride < H)) return fail(DLB_ERR_BAD_STRIDE, "a row stride of the outputs is smaller than H=%lld", (long long)H);
  if (x_row_stride < 0 || residual_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative row stride");
  NormArgs a{};
  a.x = x, a.res = residual, a.w = weight, a.y = y, a.sum = sum;
  a.rows = rows, a.x_rs = x_row_stride, a.res_rs = residual_row_stride, a.y_rs = y_row_stride, a.sum_rs = sum_row_stride;
  a.H = static_cast<int>(H), a.w_f32 = weight_dtype == kInF32, a.eps = eps;
  return launch_norm<false>(a, dtype, static_cast<hipStream_t>(stream));
}

int dlb_rms_norm_quant(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, int dtype,
                       const void* weight, int weight_dtype, void* q, float* s, int64_t s_stride_m, int64_t s_stride_k,
                       void* sum, int64_t sum_row_stride, int64_t rows, int64_t H, float eps, float quant_eps, void* stream) {
  using namespace dlb;
  clear_error();
  if (int rc = check_norm(x, residual, dtype, weight, weight_dtype, sum, rows, H)) return rc;
  if (H % kScaleBlock != 0) return fail(DLB_ERR_BAD_SHAPE, "H=%lld is not a multiple of the group size 128", (long long)H);
  if (!(quant_eps >= 1e-30f)) return fail(DLB_ERR_BAD_SHAPE, "quant_eps=%g is below 1e-30: a scale could not be divided by", quant_eps);
  if (rows == 0 || H == 0) return DLB_OK;
  if (!q || !s) return fail(DLB_ERR_NULL_POINTER, "q or s is NULL");
  if (misaligned(q, 8) || misaligned(s, 4)) return fail(DLB_ERR_ALIGNMENT, "q must be 8-byte, s 4-byte aligned");
  if (s_stride_m < 0 || s_stride_k < 0 || x_row_stride < 0 || residual_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative stride");
  if (residual && sum_row_stride < H) return fail(DLB_ERR_BAD_STRIDE, "row stride %lld of sum is smaller than H=%lld", (long long)sum_row_stride, (long long)H);
  NormArgs a{};
  a.x = x, a.res = residual, a.w = weight, a.sum = sum, a.q = static_cast<uint8_t*>(q), a.s = s;
  a.rows = rows, a.x_rs = x_row_stride, a.res_rs = residual_row_stride, a.sum_rs = sum_row_stride, a.s_sm = s_stride_m, a.s_sk = s_stride_k;
  a.H = static_cast<int>(H), a.w_f32 = weight_dtype == kInF32, a.eps = eps, a.qeps = quant_eps;
  return launch_norm<true>(a, dtype, static_cast<hipStream_t>(stream));
}

size_t dlb_rms_norm_backward_workspace_bytes(int64_t rows, int64_t H) {
  return rows > 0 && H > 0 ? static_cast<size_t>(dlb::norm_grad_shares(rows, H)) * H * sizeof(float) : 0;
}

int dlb_rms_norm_backward(const void* dy, int64_t dy_row_stride, const void* dsum, int64_t dsum_row_stride, const void* h,
                          int64_t h_row_stride, int dtype, const void* weight, int weight_dtype, void* dx, int64_t dx_row_stride,
                          void* dw, int64_t rows, int64_t H, float eps, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dlb;
  clear_error();
  if (int rc = check_norm(h, dsum, dtype, weight, weight_dtype, dsum, rows, H)) return rc;
  if (H == 0 || (rows == 0 && !dw)) return DLB_OK;
  if (dw && off_elements(dw, weight_dtype)) return fail(DLB_ERR_ALIGNMENT, "dw is not aligned to its elements");
  if (rows > 0) {
    if (!dy || !dx) return fail(DLB_ERR_NULL_POINTER, "dy or dx is NULL");
    if (off_elements(dy, dtype) || off_elements(dx, dtype)) return fail(DLB_ERR_ALIGNMENT, "a tensor is not aligned to its elements");
    if (dx_row_stride < H) return fail(DLB_ERR_BAD_STRIDE, "row stride %lld of dx is smaller than H=%lld", (long long)dx_row_stride, (long long)H);
    if (dy_row_stride < 0 || dsum_row_stride < 0 || h_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative row stride");
    const size_t need = dlb_rms_norm_backward_workspace_bytes(rows, H);
    if (dw && (!workspace || workspace_bytes < need))
      return fail(DLB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (dw && misaligned(workspace, 4)) return fail(DLB_ERR_ALIGNMENT, "workspace must be 4-byte aligned");
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int shares = norm_grad_shares(rows, H);
  if (rows > 0) {
    NormGradArgs a{};
    a.dy = dy, a.dsum = dsum, a.h = h, a.w = weight, a.dx = dx, a.dw_part = dw ? static_cast<float*>(workspace) : nullptr;
    a.rows = rows, a.dy_rs = dy_row_stride, a.dsum_rs = dsum_row_stride, a.h_rs = h_row_stride, a.dx_rs = dx_row_stride;
    a.H = static_cast<int>(H), a.w_f32 = weight_dtype == kInF32, a.eps = eps;
    const auto launch = [&](auto t, auto ds, auto whole, auto c, auto lanes, int grid, int threads, int beside) {
      hipLaunchKernelGGL((rms_norm_backward_kernel<t(), ds(), whole(), c(), lanes()>), dim3(grid), dim3(threads, beside), 0, st, a);
    };
    with_type(dtype, [&](auto t) {
      with_flag(dsum != nullptr, [&](auto ds) {
        if (H % 8 == 0) {
          constexpr std::true_type whole;
          if (with_lanes(H, [&](auto lanes) { launch(t, ds, whole, kOne, lanes, shares / (kNarrowThreads / 64), lanes(), kNarrowThreads / lanes()); })) return;
        }
        // Two workgroups of up to 512 threads fit a CU beside each other at these registers.  One and two chunks a thread, 4096 rows: of 4096
        // columns in 16 bits 24 and 29 us, of 5120 44 and 35, of 7168 64 and 51; of 4096 in fp32 40 and 47, of 8192 in fp32 90 and 97.
        const RowShape shape = row_shape(H, dtype != kInF32 && H > 4096 ? 2 : 1);
        with_flag(H % 8 == 0, [&](auto whole) {
          with_chunks<1, 2, 4>(shape.chunks, [&](auto c) { launch(t, ds, whole, c, kWave, shares, shape.threads, 1); });
        });
      });
    });
    if (int rc = finish("rms_norm_backward")) return rc;
  }
  if (!dw) return DLB_OK;
  const NormDwArgs d{static_cast<const float*>(workspace), dw, shares, static_cast<int>(H), weight_dtype};
  hipLaunchKernelGGL(rms_norm_dw_kernel, dim3(static_cast<unsigned>(ceil_div(H, 64))), dim3(64 * kDwWaves), 0, st, d);
  return finish("rms_norm_backward (dw)");
}

size_t dlb_moe_permute_workspace_bytes(int64_t tokens, int64_t topk, int64_t experts) {
  if (tokens <= 0 || topk <= 0 || experts <= 0) return 0;
  const int64_t blocks = dlb::sort_blocks(tokens * topk);
  return blocks > 1 ? static_cast<size_t>(dlb::sort_scans(blocks, experts) ? blocks + 1 : blocks) * experts * sizeof(int32_t) : 0;
}

int dlb_moe_permute(const void* ids, int ids_dtype, int64_t ids_stride_m, int64_t ids_stride_k, const void* x, int64_t x_row_stride,
                    int dtype, const float* x_s, int64_t xs_stride_m, int64_t xs_stride_k, int32_t* row_index, int32_t* source,
                    int32_t* m_indices, int32_t* row_start, int32_t* row_end, void* rows, float* rows_s, int64_t tokens, int64_t H,
                    int64_t topk, int64_t experts, int64_t alignment, int64_t num_rows, void* workspace, size_t workspace_bytes,
                    void* stream) {
  using namespace dlb;
  clear_error();
  const bool f8 = dtype == DLB_ROWS_E4M3;
  if (ids_dtype != DLB_IDX_I32 && ids_dtype != DLB_IDX_I64) return fail(DLB_ERR_BAD_DTYPE, "ids_dtype %d is not DLB_IDX_I32 / I64", ids_dtype);
  if (!f8 && bad_dtype(dtype)) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16 / F32 / DLB_ROWS_E4M3", dtype);
  if (int rc = check_rows(tokens, H, topk, num_rows)) return rc;
  if (f8 && H % kScaleBlock != 0) return fail(DLB_ERR_BAD_SHAPE, "H=%lld is not a multiple of 128", (long long)H);
  if (experts < 1 || experts > kSortMaxExperts) return fail(DLB_ERR_BAD_SHAPE, "experts=%lld is not 1 ... %d", (long long)experts, kSortMaxExperts);
  if (alignment < 1 || alignment > (1 << 20)) return fail(DLB_ERR_BAD_SHAPE, "alignment=%lld is not 1 ... 2^20", (long long)alignment);
  if (ids_stride_m < 0 || ids_stride_k < 0 || x_row_stride < 0 || xs_stride_m < 0 || xs_stride_k < 0) return fail(DLB_ERR_BAD_STRIDE, "negative stride");
  if ((tokens > 0 && (!ids || !row_index)) || (num_rows > 0 && (!source || !m_indices)) || !row_start || !row_end)
    return fail(DLB_ERR_NULL_POINTER, "ids or a table is NULL");
  if (misaligned(ids, ids_dtype == DLB_IDX_I64 ? 8 : 4) || misaligned(row_index, 4) || misaligned(source, 4) || misaligned(m_indices, 4) ||
      misaligned(row_start, 4) || misaligned(row_end, 4))
    return fail(DLB_ERR_ALIGNMENT, "ids or a table is not aligned to its elements");
  const bool copies = num_rows > 0 && H > 0;
  if (copies && (!rows || (tokens > 0 && !x))) return fail(DLB_ERR_NULL_POINTER, "x or rows is NULL");
  if (copies && f8 && (!rows_s || (tokens > 0 && !x_s))) return fail(DLB_ERR_NULL_POINTER, "e4m3 rows without their scales");
  if (f8 ? misaligned(x, 16) || misaligned(rows, 16) || x_row_stride % 16 != 0 || misaligned(x_s, 4) || misaligned(rows_s, 4)
         : off_elements(x, dtype) || off_elements(rows, dtype))
    return fail(DLB_ERR_ALIGNMENT, "x or rows is not aligned to its elements, or e4m3 rows not to 16 bytes");
  const size_t need = dlb_moe_permute_workspace_bytes(tokens, topk, experts);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(DLB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  if (need > 0 && misaligned(workspace, 4)) return fail(DLB_ERR_ALIGNMENT, "workspace must be 4-byte aligned");

  SortArgs a{};
  a.ids = ids, a.row_index = row_index, a.source = source, a.m_indices = m_indices, a.row_start = row_start, a.row_end = row_end;
  a.hist = static_cast<int32_t*>(workspace);
  a.ids_s0 = ids_stride_m, a.ids_s1 = ids_stride_k, a.n = tokens * topk, a.R = num_rows;
  a.ids_is64 = ids_dtype == DLB_IDX_I64, a.E = static_cast<int>(experts), a.topk = static_cast<int>(topk), a.align = static_cast<int>(alignment);
  SortCopyArgs c{};
  if (copies) {
    const int esz = f8 ? 1 : static_cast<int>(size_of(dtype));
    c.x = static_cast<const char*>(x), c.rows = static_cast<char*>(rows), c.row_index = row_index, c.source = source;
    if (f8) c.xs = x_s, c.rows_s = rows_s, c.xs_s0 = xs_stride_m, c.xs_s1 = xs_stride_k, c.groups = static_cast<int>(H / kScaleBlock);
    c.x_stride = x_row_stride * esz, c.rows_stride = H * esz, c.T = tokens, c.R = num_rows;
    c.row_bytes = static_cast<int>(H * esz), c.esz = esz, c.topk = static_cast<int>(topk);
    // a wave holds kSortCopyChunks KB of a row; parts down to one KB while there are fewer waves than the chip takes at once
    const int64_t kbytes = ceil_div(c.row_bytes, 1024);
    int64_t part = kSortCopyChunks;
    while (part > 1 && tokens * ceil_div(kbytes, part) < 8192) part /= 2;
    c.parts = static_cast<int>(ceil_div(kbytes, part)), c.part_bytes = static_cast<int>(part * 1024);
  }
  const bool whole_rows = c.row_bytes % 16 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t lds = (static_cast<size_t>(3) * a.E + 1) * sizeof(int) + static_cast<size_t>(16) * a.E * sizeof(uint16_t);

  if (copies && a.n <= kSortBlockSlots) {
    // 1024 slots, as many as one workgroup finds the rows of: one launch, 512 x 2 slots x 4096 bf16 6.6 us, 128 x 8 x 7168 among 256 experts
    // 10.7, 16 x 8 x 7168 among 32 5.2.  One token more, in three launches: 513 x 2 10.0 us, 129 x 8 13.6.
    const int threads = a.n <= 256 ? 256 : kSortThreads;
    const int64_t want = ceil_div(std::max(tokens * c.parts, num_rows), threads / 64), most = 512 * (kSortThreads / threads);
    const dim3 grid(static_cast<unsigned>(want < most ? want : most));
    with_flag(whole_rows, [&](auto whole) {
      hipLaunchKernelGGL((moe_sort_rows_kernel<true, whole()>), grid, dim3(threads), lds + threads * sizeof(int), st, a, 1, false, c);
    });
    return finish("moe_permute");
  }
  const int64_t blocks = sort_blocks(a.n);
  const bool summed = sort_scans(blocks, a.E);
  if (blocks > 1) {
    hipLaunchKernelGGL(moe_sort_count_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kSortThreads), static_cast<size_t>(a.E) * sizeof(int), st, a);
    if (int rc = finish("moe_permute (count)")) return rc;
    if (summed) {
      hipLaunchKernelGGL(moe_sort_scan_kernel, dim3(static_cast<unsigned>(ceil_div(a.E, 64))), dim3(64 * kScanWaves), 0, st, a, static_cast<int>(blocks));
      if (int rc = finish("moe_permute (scan)")) return rc;
    }
  }
  // further workgroups where the tables by row are longer than those by slot
  int64_t grid = ceil_div(num_rows, 4 * kSortThreads);
  if (grid > 256) grid = 256;
  if (grid < blocks) grid = blocks;
  hipLaunchKernelGGL((moe_sort_rows_kernel<false, true>), dim3(static_cast<unsigned>(grid)), dim3(kSortThreads), lds, st, a, static_cast<int>(blocks), summed, c);
  if (int rc = finish("moe_permute (tables)")) return rc;
  if (!copies) return DLB_OK;
  constexpr int kWaves = kSortCopyThreads / 64;
  c.token_blocks = static_cast<int>(std::min<int64_t>(ceil_div(tokens * c.parts, kWaves), 16384));
  c.zero_blocks = static_cast<int>(std::min<int64_t>(ceil_div(num_rows, kWaves), 1024));
  with_flag(whole_rows, [&](auto whole) {
    hipLaunchKernelGGL(moe_sort_copy_kernel<whole()>, dim3(c.token_blocks + c.zero_blocks), dim3(kSortCopyThreads), 0, st, c);
  });
  return finish("moe_permute (copy)");
}

int dlb_moe_unpermute(const void* rows, int64_t rows_row_stride, int dtype, const int32_t* row_index, const float* weights, void* out,
                      int64_t out_row_stride, int64_t tokens, int64_t H, int64_t topk, int64_t num_rows, void* stream) {
  using namespace dlb;
  clear_error();
  if (bad_dtype(dtype)) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16 / F32", dtype);
  if (int rc = check_rows(tokens, H, topk, num_rows)) return rc;
  if (tokens == 0 || H == 0) return DLB_OK;
  if (!out || !row_index || (num_rows > 0 && !rows)) return fail(DLB_ERR_NULL_POINTER, "rows, row_index or out is NULL");
  if (out_row_stride < H) return fail(DLB_ERR_BAD_STRIDE, "row stride %lld of out is smaller than H=%lld", (long long)out_row_stride, (long long)H);
  if (rows_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative row stride");
  if (off_elements(rows, dtype) || off_elements(out, dtype) || misaligned(row_index, 4) || misaligned(weights, 4))
    return fail(DLB_ERR_ALIGNMENT, "a tensor is not aligned to its elements");
  const UnpermuteArgs a{rows, row_index, weights, out, rows_row_stride, out_row_stride, tokens, num_rows, static_cast<int>(H), static_cast<int>(topk)};
  int64_t parts = ceil_div(H, 512);
  if (parts > 64) parts = 64;
  const dim3 rows_grid = row_grid(tokens), grid(rows_grid.x, static_cast<unsigned>(parts), rows_grid.y);
  with_type(dtype, [&](auto t) {
    with_flag(H % 8 == 0, [&](auto whole) { hipLaunchKernelGGL((moe_unpermute_kernel<t(), whole()>), grid, dim3(64), 0, static_cast<hipStream_t>(stream), a); });
  });
  return finish("moe_unpermute");
}

int dlb_moe_unpermute_backward(const void* dout, int64_t dout_row_stride, const void* rows, int64_t rows_row_stride, int dtype,
                               const int32_t* row_index, const int32_t* source, const float* weights, void* drows,
                               int64_t drows_row_stride, float* dweights, int64_t tokens, int64_t H, int64_t topk, int64_t num_rows,
                               void* stream) {
  using namespace dlb;
  clear_error();
  if (bad_dtype(dtype)) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16 / F32", dtype);
  if (int rc = check_rows(tokens, H, topk, num_rows)) return rc;
  if (H < 1 || H > DLB_NORM_MAX_COLUMNS) return fail(DLB_ERR_BAD_SHAPE, "H=%lld is not 1 ... %d", (long long)H, DLB_NORM_MAX_COLUMNS);
  if (tokens == 0 && num_rows == 0) return DLB_OK;
  if ((tokens > 0 && (!dout || !row_index)) || (num_rows > 0 && (!drows || !source || (dweights && !rows))))
    return fail(DLB_ERR_NULL_POINTER, "a tensor pointer is NULL");
  if (drows_row_stride < H) return fail(DLB_ERR_BAD_STRIDE, "row stride %lld of drows is smaller than H=%lld", (long long)drows_row_stride, (long long)H);
  if (dout_row_stride < 0 || rows_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative row stride");
  if (off_elements(dout, dtype) || off_elements(rows, dtype) || off_elements(drows, dtype) || misaligned(row_index, 4) || misaligned(source, 4) ||
      misaligned(weights, 4) || misaligned(dweights, 4))
    return fail(DLB_ERR_ALIGNMENT, "a tensor is not aligned to its elements");
  UnpermuteGradArgs a{};
  a.dout = dout, a.rows = rows, a.row_index = row_index, a.source = source, a.w = weights, a.drows = drows, a.dw = dweights;
  a.dout_rs = dout_row_stride, a.rows_rs = rows_row_stride, a.drows_rs = drows_row_stride;
  a.T = tokens, a.R = num_rows, a.H = static_cast<int>(H), a.topk = static_cast<int>(topk);
  a.zero_blocks = static_cast<int>(num_rows < 1024 ? num_rows : 1024);
  const RowShape shape = row_shape(H, 2);  // 4096 tokens of 7168 x 8 rows: one chunk a thread 219 us, two 195, four 197
  const int64_t grid = tokens + a.zero_blocks;
  with_type(dtype, [&](auto t) {
    with_flag(dweights != nullptr, [&](auto dw) {
      with_flag(H % 8 == 0, [&](auto whole) {
        with_chunks<1, 2, 4>(shape.chunks, [&](auto c) {
          hipLaunchKernelGGL((moe_unpermute_backward_kernel<t(), dw(), whole(), c()>), row_grid(grid), dim3(shape.threads), 0,
                             static_cast<hipStream_t>(stream), a);
        });
      });
    });
  });
  return finish("moe_unpermute_backward");
}

size_t dlb_w4_gemm_workspace_bytes(int64_t rows, int64_t N, int64_t K, int64_t experts) {
  if (experts != 0 || rows <= 0 || N <= 0 || K <= 0) return 0;
  const dlb::W4Plan plan = dlb::w4_plan(rows, false, 1, N, K);
  return plan.slices > 1 ? static_cast<size_t>(plan.slices) * rows * N * sizeof(float) : 0;
}

int dlb_w4_gemm(const void* x, int64_t x_row_stride, int dtype, const void* q, const void* s, int s_dtype, const void* z, void* y,
                int64_t y_row_stride, const int32_t* row_start, const int32_t* row_end, int64_t rows, int64_t N, int64_t K,
                int64_t group, int64_t experts, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dlb;
  clear_error();
  if (dtype != kInBf16 && dtype != kInF16) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16", dtype);
  if (s_dtype != kInBf16 && s_dtype != kInF16) return fail(DLB_ERR_BAD_DTYPE, "s_dtype %d is not DLB_IN_BF16 / F16", s_dtype);
  if (rows < 0 || N < 0 || K < 0 || experts < 0)
    return fail(DLB_ERR_BAD_SHAPE, "negative dimension (rows=%lld N=%lld K=%lld experts=%lld)", (long long)rows, (long long)N, (long long)K, (long long)experts);
  if (group != 32 && group != 64 && group != 128) return fail(DLB_ERR_BAD_SHAPE, "group=%lld is not 32, 64 or 128", (long long)group);
  if (K % group != 0) return fail(DLB_ERR_BAD_SHAPE, "K=%lld is not a multiple of the group size %lld", (long long)K, (long long)group);
  if (!row_start != !row_end) return fail(DLB_ERR_NULL_POINTER, "row_start and row_end come together");
  if (!row_start && experts != 1) return fail(DLB_ERR_BAD_SHAPE, "%lld experts without row ranges", (long long)experts);
  if (rows > (1ll << 31) - 1 || N > (1ll << 27) || K > (1ll << 30) || experts > (1 << 20))
    return fail(DLB_ERR_BAD_SHAPE, "rows=%lld / N=%lld / K=%lld / experts=%lld beyond the supported range", (long long)rows, (long long)N, (long long)K,
                (long long)experts);
  if (rows == 0 || N == 0 || experts == 0) return DLB_OK;
  if (K == 0) return fail(DLB_ERR_BAD_SHAPE, "K=0: there is no product");
  if (!x || !q || !s || !y) return fail(DLB_ERR_NULL_POINTER, "x, q, s or y is NULL");
  if (x_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative row stride");
  if (y_row_stride < N) return fail(DLB_ERR_BAD_STRIDE, "row stride %lld of y is smaller than N=%lld", (long long)y_row_stride, (long long)N);
  // a tile is one buffer of 32-bit offsets
  if (x_row_stride > (1 << 24) || K > (1 << 24)) return fail(DLB_ERR_BAD_STRIDE, "x row stride %lld / K=%lld beyond 2^24", (long long)x_row_stride, (long long)K);
  if (misaligned(q, 16) || misaligned(x, 4) || x_row_stride % 2 != 0 || off_elements(y, dtype) || off_elements(s, s_dtype) || misaligned(row_start, 4) ||
      misaligned(row_end, 4))
    return fail(DLB_ERR_ALIGNMENT, "q must be 16-byte, rows of x 4-byte aligned, the others to their elements");
  W4Args a{};
  a.x = x, a.q = static_cast<const uint8_t*>(q), a.s = s, a.z = static_cast<const uint8_t*>(z), a.y = y, a.row_start = row_start, a.row_end = row_end;
  a.x_rs = x_row_stride, a.y_rs = y_row_stride, a.rows = rows;
  a.N = static_cast<int>(N), a.K = static_cast<int>(K), a.G = static_cast<int>(K / group), a.E = static_cast<int>(experts), a.s_type = s_dtype;
  a.q_es = N * (K / 2), a.s_es = N * a.G;
  const int64_t busy = experts < rows ? experts : rows;  // experts that can have a row
  const W4Plan plan = row_start ? w4_plan(ceil_div(rows, busy), true, busy, N, K) : w4_plan(rows, false, 1, N, K);
  const int64_t y_blocks = row_start ? busy : ceil_div(rows, 16 * plan.mt);
  if (y_blocks > 65535) return fail(DLB_ERR_BAD_SHAPE, "rows=%lld / experts=%lld beyond the supported range", (long long)rows, (long long)experts);
  const size_t need = plan.slices > 1 ? static_cast<size_t>(plan.slices) * rows * N * sizeof(float) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(DLB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  if (need > 0 && misaligned(workspace, 4)) return fail(DLB_ERR_ALIGNMENT, "workspace must be 4-byte aligned");
  if (ceil_div(rows * N, 256) > (1ll << 31) - 1) return fail(DLB_ERR_BAD_SHAPE, "rows=%lld x N=%lld beyond the supported range", (long long)rows, (long long)N);
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* const sums = static_cast<float*>(workspace);
  const auto launch = [&](auto t, auto zeros) {
    if (group == 128)
      launch_w4<t(), 1, zeros()>(a, plan, y_blocks, sums, st);
    else if (group == 64)
      launch_w4<t(), 2, zeros()>(a, plan, y_blocks, sums, st);
    else
      launch_w4<t(), 4, zeros()>(a, plan, y_blocks, sums, st);
  };
  const auto with_zeros = [&](auto t) { z ? launch(t, std::true_type()) : launch(t, std::false_type()); };
  if (dtype == kInBf16)
    with_zeros(std::integral_constant<int, kInBf16>());
  else
    with_zeros(std::integral_constant<int, kInF16>());
  return finish("w4_gemm");
}

int dlb_w4_quant(const void* w, int64_t w_row_stride, int dtype, void* q, void* s, void* z, int64_t rows, int64_t K, int64_t group,
                 void* stream) {
  using namespace dlb;
  clear_error();
  if (dtype != kInBf16 && dtype != kInF16) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16, the types of scales", dtype);
  if (rows < 0 || K < 0) return fail(DLB_ERR_BAD_SHAPE, "negative dimension (rows=%lld K=%lld)", (long long)rows, (long long)K);
  if (group != 32 && group != 64 && group != 128) return fail(DLB_ERR_BAD_SHAPE, "group=%lld is not 32, 64 or 128", (long long)group);
  if (K % group != 0) return fail(DLB_ERR_BAD_SHAPE, "K=%lld is not a multiple of the group size %lld", (long long)K, (long long)group);
  if (K > (1ll << 28)) return fail(DLB_ERR_BAD_SHAPE, "K=%lld beyond the supported range", (long long)K);
  if (rows == 0 || K == 0) return DLB_OK;
  if (!w || !q || !s) return fail(DLB_ERR_NULL_POINTER, "w, q or s is NULL");
  if (w_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative row stride");
  if (off_elements(w, dtype) || off_elements(s, dtype) || misaligned(q, 4)) return fail(DLB_ERR_ALIGNMENT, "w and s must be aligned to their elements, q to 4 bytes");
  const W4QuantArgs a{w, static_cast<uint8_t*>(q), s, static_cast<uint8_t*>(z), rows, w_row_stride, static_cast<int>(K / group), static_cast<int>(group)};
  const int64_t blocks = ceil_div(rows * a.G * (group / 8), 256);
  const dim3 grid(static_cast<unsigned>(blocks < 8192 ? blocks : 8192));
  const auto launch = [&](auto t) { hipLaunchKernelGGL(w4_quant_kernel<t()>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a); };
  dtype == kInBf16 ? launch(std::integral_constant<int, kInBf16>()) : launch(std::integral_constant<int, kInF16>());
  return finish("w4_quant");
}

}  // extern "C"
