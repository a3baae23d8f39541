// Host-side helpers of the entry points: the end of a launch, runtime values as template arguments, grids of rows.
#pragma once

#include <algorithm>
#include <type_traits>

#include "../../include/dlblas_fp8_gemm.h"
#include "host_common.h"
#include "rows.h"

namespace dlb {

inline int finish(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(DLB_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return DLB_OK;
}

inline bool bad_dtype(int d) { return d < kInBf16 || d > kInF32; }
inline int64_t size_of(int d) { return d == kInF32 ? 4 : 2; }
inline bool off_elements(const void* p, int dtype) { return misaligned(p, size_of(dtype)); }

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

// A grid of `blocks` workgroups in two dimensions.
inline dim3 row_grid(int64_t blocks) {
  constexpr int64_t kMost = 1 << 21;  // of up to 1024 threads, of which one dimension holds fewer than 2^32
  return dim3(static_cast<unsigned>(std::min(blocks, kMost)), static_cast<unsigned>(ceil_div(blocks, kMost)));
}

}  // namespace dlb
