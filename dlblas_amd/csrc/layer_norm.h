// Layer norm with the residual's addition and its gradient, for gfx950.
//
//   h = x + res rounded to the rows' type (without a residual h = x),  m = mean(h),  r = 1 / sqrt(mean((h - m)^2) + eps),  n = (h - m) r,
//   y = n w + b
//   gradient:  t = w dy,  dh = r (t - mean(t) - n mean(t n)) + dsum,  dw = sum over the rows of dy n,  db = sum over the rows of dy
//
// h is rounded before the norm reads it, as in the RMS norm and for the same reason; everything else is fp32 with one rounding at the store.  The
// squares are those of h - m, from a second sweep over the registers: the difference of mean(h^2) and m^2 would lose a row whose mean is large
// against its spread.  The same sweep has the sum of h - m, what the rounded mean is off by: corrected by it the mean of a constant row is its value, which the sum's and
// 1 / H's roundings miss (7168 columns of 1e5 in bf16 by 2^-7, more than sqrt(eps)).  Sums of h are taken by 2^-16 and h - m by half, both exact, so that neither leaves the range where h is finite.  m and r of every row are kept for the gradient (8 bytes a row), which then needs one pass of sums over the workgroup
// instead of three.
//
// Bound by memory like the RMS norm, and built like it: a row is read once into registers (8 elements a chunk, CH chunks a thread) and the results
// leave from there; rows of up to 16 or 32 chunks share waves.
#pragma once

#include "rms_norm.h"

namespace dlb {

struct LayerNormArgs {
  const void* x;
  const void* res;   // or NULL
  const void* w;     // [H], the rows' type or fp32
  const void* b;     // the same, or NULL
  void* y;
  void* sum;         // h, with a residual
  float* stats;      // [rows][2]: m and r, or NULL: not wanted
  int64_t rows, x_rs, res_rs, y_rs, sum_rs;
  int H;
  int w_f32;
  float eps;
};

// Where rows end: on a chunk; inside one, whose lane takes the last eight columns instead, some of them a second time, which it leaves out of the sums and stores as the
// lane in front does; or in front of the first chunk's end, and elements are loaded one by one.  (Behind a branch for the last chunk rows that are asked for ahead
// would be waited for at once: 16384 x 2050 bf16, the gradient, 129 us.)
enum Edge { kOnChunk, kInChunk, kBelowChunk };

// Sum over the threads of a row.  `part`: a set of its own for each sum between two barriers.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* part, int tid, int threads) {
  v = wave_sum<LANES>(v);
  if (LANES < 64 || threads == 64) return v;
  if ((tid & 63) == 0) part[tid >> 6] = v;
  lds_barrier();
  v = 0.f;
  for (int i = 0; i < threads / 64; ++i) v += part[i];
  return v;
}

// The same of two.
template <int LANES>
__device__ __forceinline__ void row_sums(float& a, float& b, float* part_a, float* part_b, int tid, int threads) {
  a = wave_sum<LANES>(a), b = wave_sum<LANES>(b);
  if (LANES < 64 || threads == 64) return;
  if ((tid & 63) == 0) part_a[tid >> 6] = a, part_b[tid >> 6] = b;
  lds_barrier();
  a = b = 0.f;
  for (int i = 0; i < threads / 64; ++i) a += part_a[i], b += part_b[i];
}

// One workgroup per row, or blockDim.y narrow rows, as in rms_norm_kernel.
template <int T, bool RES, Edge EDGE, int CH, int LANES>
__global__ void __launch_bounds__(kNormMaxThreads) layer_norm_kernel(const LayerNormArgs p) {
  constexpr bool WHOLE = EDGE != kBelowChunk;
  __shared__ float part[3][kNormMaxWaves];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int64_t row = grid_row() * blockDim.y + beside<LANES>();
  if (row >= p.rows) return;  // with rows beside each other in a workgroup there is no barrier
  const int chunks = (p.H + 7) / 8;
  int at[CH], again[CH];  // the first column of a lane's chunk, how many of it the lane in front has
  Raw8 h[CH], res[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = 8 * min(c * threads + tid, chunks - 1);
    at[c] = EDGE == kInChunk ? min(i, p.H - 8) : i, again[c] = i - at[c];
    h[c] = load_raw8<T, WHOLE>(p.x, row * p.x_rs, at[c], p.H);
    if (RES) res[c] = load_raw8<T, WHOLE>(p.res, row * p.res_rs, at[c], p.H);
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
      if (c * threads + tid < chunks) store_raw8<T, WHOLE>(p.sum, row * p.sum_rs, at[c], h[c], p.H);
    }
  }
  const float inv_h = 1.0f / static_cast<float>(p.H);
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float v[8], e = 0.f;
    quant_unpack8<T>(h[c], v);
#pragma unroll
    for (int k = 0; k < 8; ++k) e = fmaf(EDGE == kInChunk && k < again[c] ? 0.f : v[k], 0x1p-16f, e);  // elements past the end are zero
    s += c * threads + tid < chunks ? e : 0.f;
  }
  const float near = row_sum<LANES>(s, part[0], tid, threads) * (0x1p16f * inv_h), rough = 0.5f * near;
  s = 0.f;
  float left = 0.f;  // of (h - near) / 2, by 2^-16 as above
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float v[8], e = 0.f, l = 0.f;
    quant_unpack8<T>(h[c], v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float d = (EDGE == kInChunk && k < again[c]) || (EDGE == kBelowChunk && k >= p.H) ? 0.f : fmaf(v[k], 0.5f, -rough);
      e = fmaf(d, d, e), l = fmaf(d, 0x1p-16f, l);
    }
    s += c * threads + tid < chunks ? e : 0.f, left += c * threads + tid < chunks ? l : 0.f;
  }
  row_sums<LANES>(s, left, part[1], part[2], tid, threads);
  const float off = left * (0x1p16f * inv_h);  // half of what `near` is off by
  const float mean = fmaf(2.0f, off, near), half = 0.5f * mean;
  // (one rounding, so that squares beyond the range stay beyond it; NaN comes back by the mean)
  const float r = 1.0f / sqrtf(fmaxf(4.0f * fmaf(-off, off, s * inv_h), 0.f) + p.eps), twice = 2.0f * r;
  if (p.stats && tid == 0) p.stats[2 * row] = mean, p.stats[2 * row + 1] = r;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (c * threads + tid >= chunks) continue;
    float v[8], w[8], b[8];
    quant_unpack8<T>(h[c], v);
    load_weight8<T, WHOLE>(p.w, p.w_f32, at[c], p.H, w);
    if (p.b) {
      load_weight8<T, WHOLE>(p.b, p.w_f32, at[c], p.H, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = fmaf(fmaf(v[k], 0.5f, -half) * twice, w[k], b[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = fmaf(v[k], 0.5f, -half) * twice * w[k];
    }
    store_raw8<T, WHOLE>(p.y, row * p.y_rs, at[c], pack_raw8<T>(v), p.H);
  }
}

struct LayerNormGradArgs {
  const void* dy;
  const void* dsum;    // or NULL: gradient of h by its other use
  const void* h;
  const void* w;
  const float* stats;  // [rows][2]
  void* dx;
  float* part;         // [shares][columns] or NULL: sums over the rows of a workgroup (of narrow rows: a wave) for dw, behind them those for db
  int64_t rows, dy_rs, dsum_rs, h_rs, dx_rs;
  int H, columns;      // columns: H, or 2 H with those for db
  int w_f32;
};

// Workers, shares, rows asked for ahead: as in rms_norm_backward_kernel.
template <int T, bool DSUM, bool BIAS, Edge EDGE, int CH, int LANES>
__global__ void __launch_bounds__(kNormMaxThreads) layer_norm_backward_kernel(const LayerNormGradArgs p) {
  constexpr bool WHOLE = EDGE != kBelowChunk, kAhead = CH == 1 || (CH == 2 && T != kInF32);
  __shared__ float part[2][2][kNormMaxWaves];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int worker = blockIdx.x * blockDim.y + beside<LANES>(), workers = gridDim.x * blockDim.y;
  const int chunks = (p.H + 7) / 8;
  const float inv_h = 1.0f / static_cast<float>(p.H);
  float dw[CH][8], db[BIAS ? CH : 1][8];
  int at[CH], again[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = 8 * min(c * threads + tid, chunks - 1);
    at[c] = EDGE == kInChunk ? min(i, p.H - 8) : i, again[c] = i - at[c];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      dw[c][k] = 0.f;
      if (BIAS) db[c][k] = 0.f;
    }
  }
  struct Row {
    Raw8 dy[CH], h[CH], ds[CH];
    float mean, r;
  };
  auto load = [&](int64_t row, Row& r) {
    r.mean = p.stats[2 * row], r.r = p.stats[2 * row + 1];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      r.h[c] = load_raw8<T, WHOLE>(p.h, row * p.h_rs, at[c], p.H);
      r.dy[c] = load_raw8<T, WHOLE>(p.dy, row * p.dy_rs, at[c], p.H);
      if (DSUM && CH < 4) r.ds[c] = load_raw8<T, WHOLE>(p.dsum, row * p.dsum_rs, at[c], p.H);
    }
  };
  // The weights stay in registers where rows are asked for ahead: loads return in order, so a weight that is loaded behind the next row waits for that row.
  float kept[kAhead ? CH : 1][8];
  if (kAhead) {
#pragma unroll
    for (int c = 0; c < CH; ++c) load_weight8<T, WHOLE>(p.w, p.w_f32, at[c], p.H, kept[c]);
  }
  const auto weights = [&](int c, float(&w)[8]) {
    if (!kAhead) return load_weight8<T, WHOLE>(p.w, p.w_f32, at[c], p.H, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = kept[c][k];
  };
  Row now, next;
  if (kAhead) load(min(static_cast<int64_t>(worker), p.rows - 1), now);
  int turn = 0;
  for (int64_t row = worker; row < p.rows; row += workers, turn ^= 1) {
    if (kAhead)
      load(min(row + workers, p.rows - 1), next);  // behind the last row that one again
    else
      load(row, now);
    const float half = 0.5f * now.mean, r = now.r, twice = 2.0f * r;
    float sum = 0.f, dot = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float hv[8], g[8], w[8], s = 0.f, d = 0.f;
      quant_unpack8<T>(now.h[c], hv);
      quant_unpack8<T>(now.dy[c], g);
      weights(c, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // elements past the end: g is zero
        const float t = EDGE == kInChunk && k < again[c] ? 0.f : g[k] * w[k];
        s += t;
        d = fmaf(t, fmaf(hv[k], 0.5f, -half) * twice, d);
      }
      const bool live = c * threads + tid < chunks;
      sum += live ? s : 0.f, dot += live ? d : 0.f;
      if (CH == 4) __builtin_amdgcn_sched_barrier(0);  // four chunks fill the registers: one chunk's weights at a time
    }
    sum = wave_sum<LANES>(sum), dot = wave_sum<LANES>(dot);
    if (LANES == 64 && threads > 64) {
      // two sets of sums in turn: a wave may be one row ahead of the others, never two
      if ((tid & 63) == 0) part[turn][0][tid >> 6] = sum, part[turn][1][tid >> 6] = dot;
      lds_barrier();
      sum = dot = 0.f;
      for (int i = 0; i < threads / 64; ++i) sum += part[turn][0][i], dot += part[turn][1][i];
    }
    const float middle = sum * inv_h, along = dot * inv_h;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float hv[8], g[8], w[8];
      quant_unpack8<T>(now.h[c], hv);
      quant_unpack8<T>(now.dy[c], g);
      weights(c, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float n = fmaf(hv[k], 0.5f, -half) * twice;
        dw[c][k] = fmaf(g[k], n, dw[c][k]);
        if (BIAS) db[c][k] += g[k];
        g[k] = r * (fmaf(g[k], w[k], -middle) - n * along);
      }
      if (DSUM) {
        float d[8];
        if (CH == 4) now.ds[c] = load_raw8<T, WHOLE>(p.dsum, row * p.dsum_rs, at[c], p.H);
        quant_unpack8<T>(now.ds[c], d);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] += d[k];
      }
      if (c * threads + tid < chunks) store_raw8<T, WHOLE>(p.dx, row * p.dx_rs, at[c], pack_raw8<T>(g), p.H);
      if (CH == 4) __builtin_amdgcn_sched_barrier(0);
    }
    if (kAhead) now = next;
  }
  if (!p.part) return;
#pragma unroll
  for (int off = LANES; off < 64; off <<= 1)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      dw[0][k] += __shfl_xor(dw[0][k], off);
      if (BIAS) db[0][k] += __shfl_xor(db[0][k], off);
    }
  if (worker % (64 / LANES) != 0) return;
  const int64_t share = static_cast<int64_t>(worker / (64 / LANES)) * p.columns;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (c * threads + tid >= chunks) continue;
    store_raw8<kInF32, WHOLE>(p.part, share, at[c], pack_raw8<kInF32>(dw[c]), p.H);
    if (BIAS) store_raw8<kInF32, WHOLE>(p.part, share + p.H, at[c], pack_raw8<kInF32>(db[c]), p.H);
  }
}

}  // namespace dlb
