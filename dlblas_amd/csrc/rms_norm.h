// Root-mean-square norm with the residual's addition, its gradient, and the form whose output is quantised 1 x 128, for gfx950.
//
//   h = x + res rounded to the rows' type (without a residual h = x),  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   quantising:  s = max(max |y|, qeps) / 448 per 128 columns,  q = e4m3(y / s); y itself is not rounded in between
//   gradient:    dh = r (w dy) - h r^3 / H sum(w dy h) + dsum,   dw = sum over the rows of dy h r
//
// h is rounded before the norm reads it: it is what the next layer adds to and what the gradient starts from, so both see the same
// rows.  Everything else is held in fp32 and rounded once at the store.  That holds for the sum of squares too: of a row whose sum passes
// 2^128 r is 0.
//
// All of it is bound by memory: a row is read once into registers (8 elements a chunk, CH chunks a thread), the sums cross the
// workgroup once, and the results leave from the registers.  Chunks are consecutive over the lanes, so 16 lanes hold a group of
// 128 columns and find its largest value among themselves.  Rows at any element boundary and widths that are no multiple of 8
// take the same path: global memory serves a 16-byte access at its element's alignment, and the last chunk of a row may be short.
#pragma once

#include "rows.h"

namespace dlb {

constexpr int kNormMaxThreads = 1024;
constexpr int kNormMaxWaves = kNormMaxThreads / 64;

struct NormArgs {
  const void* x;
  const void* res;  // or NULL
  const void* w;    // [H], the rows' type or fp32
  void* y;          // not written by the quantising form
  void* sum;        // h, with a residual
  uint8_t* q;       // quantising form: [rows][H]
  float* s;
  int64_t rows, x_rs, res_rs, y_rs, sum_rs, s_sm, s_sk;
  int H;
  int w_f32;
  float eps, qeps;
};

// The largest |y| of 16 lanes, or the largest |h w|, as bits, which put NaN above infinity: a group that holds one gets a scale that shows it.
__device__ __forceinline__ uint32_t group_max(bool hw, const float (&h)[8], const float (&w)[8], const float (&y)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(hw ? h[k] * w[k] : y[k]) & 0x7fffffffu);
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 16)));
  return top;
}

// One workgroup per row, blockDim.x = the threads that the row's chunks need at CH chunks each, or blockDim.y narrow rows
// (up to 16 or 32 chunks: LANES of a wave a row); a thread past the last chunk reads that one
// again and leaves no trace.  8192 x 7168 bf16 with residual, quantised, 413 MB: 77 us, 5.3 TB/s (a large copy reaches 5.0 here); 4096 x 7168
// with residual, not quantised, 235 MB: 40 us, 5.8 TB/s, part of it from the cache; one row 3.7 us, launch and latency.
template <int T, bool QUANT, bool RES, bool WHOLE, int CH, int LANES>
__global__ void __launch_bounds__(kNormMaxThreads) rms_norm_kernel(const NormArgs p) {
  __shared__ float part[kNormMaxWaves];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int64_t row = grid_row() * blockDim.y + beside<LANES>();
  if (row >= p.rows) return;  // with rows beside each other in a workgroup there is no barrier
  const int chunks = (p.H + 7) / 8;
  int at[CH];
  Raw8 h[CH], res[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    at[c] = min(c * threads + tid, chunks - 1);
    h[c] = load_raw8<T, WHOLE>(p.x, row * p.x_rs, 8 * at[c], p.H - 8 * at[c]);
    if (RES) res[c] = load_raw8<T, WHOLE>(p.res, row * p.res_rs, 8 * at[c], p.H - 8 * at[c]);
  }
  if (RES) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float a[8], b[8];
      quant_unpack8<T>(h[c], a);
      quant_unpack8<T>(res[c], b);
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] += b[k];
      h[c] = pack_raw8<T>(a);
      if (c * threads + tid < chunks) store_raw8<T, WHOLE>(p.sum, row * p.sum_rs, 8 * at[c], h[c], p.H - 8 * at[c]);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float v[8], s = 0.f;
    quant_unpack8<T>(h[c], v);
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(v[k], v[k], s);
    ss += c * threads + tid < chunks ? s : 0.f;
  }
  ss = wave_sum<LANES>(ss);
  if (LANES == 64 && threads > 64) {
    if ((tid & 63) == 0) part[tid >> 6] = ss;
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < threads / 64; ++i) ss += part[i];
  }
  const float r = 1.0f / sqrtf(ss / static_cast<float>(p.H) + p.eps);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = c * threads + tid;
    if (i >= chunks) continue;  // whole groups of 16 lanes: a quantised row is a multiple of 128 wide
    float v[8], w[8];
    quant_unpack8<T>(h[c], v);
    load_weight8<T, WHOLE>(p.w, p.w_f32, 8 * i, p.H - 8 * i, w);
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = v[k] * r * w[k];
    if (!QUANT) {
      store_raw8<T, WHOLE>(p.y, row * p.y_rs, 8 * i, pack_raw8<T>(y), p.H - 8 * i);
      continue;
    }
    // y / s = 448 h w / max |h w|: r cancels, and for bf16 rows and weights (8 + 8 + 3 bits) the operands of that quotient are exact, so a
    // value half way between two codes stays there (with y rounded first 1 of 10^4 codes differed, with these operands none of 3 10^6).  fp16
    // rows take 25 bits, one rounding of fp32, and fp32 weights under 16-bit rows two.
    // Rows of fp32 take y, as the quantiser does that reads it from memory, and so do groups whose h w is close to the ends of fp32.
    constexpr bool kExact = T != kInF32;
    float num[8], den;
    uint32_t top = group_max(kExact, v, w, y);
    float scale = __uint_as_float(top) * r / 448.0f;
    if (kExact && top - (27u << 23) < (200u << 23) && scale * 448.0f >= p.qeps) {  // 2^-100 to 2^100
#pragma unroll
      for (int k = 0; k < 8; ++k) num[k] = v[k] * w[k] * 448.0f;
      den = __uint_as_float(top);
    } else {
      if (kExact) top = group_max(false, v, w, y);
      const float amax = __uint_as_float(top);
      scale = den = (amax < p.qeps ? p.qeps : amax) / 448.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) num[k] = y[k];
    }
    const float inv_den = 1.0f / den;
    int packed[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = div_by_scale(num[4 * k + j], den, inv_den);  // at most 448 and a rounding: no clamp
      int word = __builtin_amdgcn_cvt_pk_fp8_f32(e[0], e[1], 0, false);
      packed[k] = __builtin_amdgcn_cvt_pk_fp8_f32(e[2], e[3], word, true);
    }
    *reinterpret_cast<v2i*>(p.q + row * p.H + 8 * i) = v2i{packed[0], packed[1]};
    if ((tid & 15) == 0) p.s[row * p.s_sm + (i >> 4) * p.s_sk] = scale;
  }
}

struct NormGradArgs {
  const void* dy;
  const void* dsum;  // or NULL: gradient of h by its other use
  const void* h;
  const void* w;
  void* dx;
  float* dw_part;    // [shares][H] or NULL: sums over the rows of a workgroup, of narrow rows those of a wave
  int64_t rows, dy_rs, dsum_rs, h_rs, dx_rs;
  int H;
  int w_f32;
  float eps;
};

// A worker takes rows worker, worker + workers, ... and keeps its share of dw in registers; the shares of all workers are
// added by rms_norm_dw_kernel in a fixed order, so the gradient is the same in every run.  The next row is on its way while the sums of
// this one cross the workgroup, where a row of two chunks a thread leaves the registers for it.  Threads past the last chunk as above.
// 4096 x 7168 bf16 with the sum's gradient, 235 MB and 15 of shares: 52 us, 4.8 TB/s; 1237 x 2050 fp32 13 us.
template <int T, bool DSUM, bool WHOLE, int CH, int LANES>
__global__ void __launch_bounds__(kNormMaxThreads) rms_norm_backward_kernel(const NormGradArgs p) {
  constexpr bool kAhead = CH == 1 || (CH == 2 && T != kInF32);
  __shared__ float part[2][2][kNormMaxWaves];
  const int tid = threadIdx.x, threads = blockDim.x;
  // workers: workgroups, or where a wave or part of one has room for a row these
  const int worker = blockIdx.x * blockDim.y + beside<LANES>(), workers = gridDim.x * blockDim.y;
  const int chunks = (p.H + 7) / 8;
  float dw[CH][8];
  int at[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    at[c] = min(c * threads + tid, chunks - 1);
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[c][k] = 0.f;
  }
  struct Row {
    Raw8 dy[CH], h[CH], ds[CH];
  };
  auto load = [&](int64_t row, Row& r) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = 8 * at[c];
      r.h[c] = load_raw8<T, WHOLE>(p.h, row * p.h_rs, col, p.H - col);
      r.dy[c] = load_raw8<T, WHOLE>(p.dy, row * p.dy_rs, col, p.H - col);
      if (DSUM && CH < 4) r.ds[c] = load_raw8<T, WHOLE>(p.dsum, row * p.dsum_rs, col, p.H - col);
    }
  };
  Row now, next;
  if (kAhead) load(min(static_cast<int64_t>(worker), p.rows - 1), now);
  int turn = 0;
  for (int64_t row = worker; row < p.rows; row += workers, turn ^= 1) {
    if (kAhead)
      load(min(row + workers, p.rows - 1), next);  // behind the last row that one again
    else
      load(row, now);
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float hv[8], g[8], w[8], s = 0.f, d = 0.f;
      quant_unpack8<T>(now.h[c], hv);
      quant_unpack8<T>(now.dy[c], g);
      load_weight8<T, WHOLE>(p.w, p.w_f32, 8 * at[c], p.H - 8 * at[c], w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        s = fmaf(hv[k], hv[k], s);
        d = fmaf(g[k] * w[k], hv[k], d);
      }
      const bool live = c * threads + tid < chunks;
      ss += live ? s : 0.f, dot += live ? d : 0.f;
      if (CH == 4) __builtin_amdgcn_sched_barrier(0);  // four chunks fill the registers: one chunk's weights at a time
    }
    ss = wave_sum<LANES>(ss), dot = wave_sum<LANES>(dot);
    if (LANES == 64 && threads > 64) {
      // two sets of sums in turn: a wave may be one row ahead of the others, never two
      if ((tid & 63) == 0) part[turn][0][tid >> 6] = ss, part[turn][1][tid >> 6] = dot;
      lds_barrier();
      ss = dot = 0.f;
      for (int i = 0; i < threads / 64; ++i) ss += part[turn][0][i], dot += part[turn][1][i];
    }
    const float r = 1.0f / sqrtf(ss / static_cast<float>(p.H) + p.eps);
    const float along = r * r * dot / static_cast<float>(p.H);  // dh = r (w dy - h along)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float hv[8], g[8], w[8];
      quant_unpack8<T>(now.h[c], hv);
      quant_unpack8<T>(now.dy[c], g);
      load_weight8<T, WHOLE>(p.w, p.w_f32, 8 * at[c], p.H - 8 * at[c], w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        dw[c][k] = fmaf(g[k], hv[k] * r, dw[c][k]);
        g[k] = r * (g[k] * w[k] - hv[k] * along);
      }
      if (DSUM) {
        float d[8];
        if (CH == 4) now.ds[c] = load_raw8<T, WHOLE>(p.dsum, row * p.dsum_rs, 8 * at[c], p.H - 8 * at[c]);
        quant_unpack8<T>(now.ds[c], d);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] += d[k];
      }
      if (c * threads + tid < chunks) store_raw8<T, WHOLE>(p.dx, row * p.dx_rs, 8 * at[c], pack_raw8<T>(g), p.H - 8 * at[c]);
      if (CH == 4) __builtin_amdgcn_sched_barrier(0);
    }
    if (kAhead) now = next;
  }
  if (!p.dw_part) return;
#pragma unroll
  for (int off = LANES; off < 64; off <<= 1)
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[0][k] += __shfl_xor(dw[0][k], off);
  if (worker % (64 / LANES) != 0) return;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = c * threads + tid;
    if (i < chunks) store_raw8<kInF32, WHOLE>(p.dw_part, static_cast<int64_t>(worker / (64 / LANES)) * p.H, 8 * i, pack_raw8<kInF32>(dw[c]), p.H - 8 * i);
  }
}

// dw[col] = sum over the parts: a wave adds every kDwWaves-th, eight sums at a time, and the waves' sums are added in pairs.  512 shares of
// 7168: 4 to 5 us (15 MB); four waves instead of sixteen 8, loads behind a branch 12.
// With db (the layer norm's) a share has its columns behind those of dw.
struct NormDwArgs {
  const float* part;
  void *dw, *db;
  int parts, H, columns, dw_type;  // columns of a share: H, or 2 H
};
constexpr int kDwWaves = 16;

__global__ void __launch_bounds__(64 * kDwWaves) rms_norm_dw_kernel(const NormDwArgs p) {
  __shared__ float sums[kDwWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + lane;
  float v[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) v[u] = 0.f;
  const float* const mine = p.part + min(col, p.columns - 1);
  for (int b = wave; b < p.parts; b += 8 * kDwWaves) {
    float e[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) e[u] = mine[static_cast<int64_t>(min(b + u * kDwWaves, p.parts - 1)) * p.columns];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] += b + u * kDwWaves < p.parts ? e[u] : 0.f;
  }
  sums[wave][lane] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  __syncthreads();
  if (wave != 0 || col >= p.columns) return;
#pragma unroll
  for (int n = kDwWaves / 2; n >= 1; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) sums[i][lane] += sums[i + n][lane];
  const float s = sums[0][lane];
  void* const to = col < p.H ? p.dw : p.db;
  const int at = col < p.H ? col : col - p.H;
  if (p.dw_type == kInF32)
    static_cast<float*>(to)[at] = s;
  else if (p.dw_type == kInBf16)
    static_cast<__bf16*>(to)[at] = static_cast<__bf16>(s);
  else
    static_cast<_Float16*>(to)[at] = static_cast<_Float16>(s);
}

}  // namespace dlb
