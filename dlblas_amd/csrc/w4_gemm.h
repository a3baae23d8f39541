// Products of a few rows with 4-bit weights and group scales for gfx950, and the quantiser that makes such weights.
//
//   y[m, n] = sum over the groups g of s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g])        z = 8 without zero points
//
// One kernel for both layouts: all rows against one matrix, or the rows [row_start[e], row_end[e]) against the matrix of expert e.
// Bound by the weights' bytes while the rows are few, so every weight byte goes from memory to a register once and straight into
// v_mfma_f32_16x16x32: a lane's 16 bytes are 32 weights of one row of the matrix, four MFMA steps.  There is no conversion: a code
// moved to the top of the significand of the float 16 is 16 + q exactly (bf16: bits 3 to 6, fp16: bits 6 to 9), a shift and an
// and-or for two weights, and the 16 leaves through the sum of x over the group, which one more MFMA with a matrix of ones gives for
// all tiles of a wave:
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x
// in fp32; the scale multiplies that once per group.  What this costs is rounding of the fp32 sums of terms up to 31 |x| instead of
// |q - z| |x|: the unit adds the 8 products of a quarter cut off 2^-24 below the largest of them and rounds after each quarter
// (measured with ladders of powers of two), so a group's sum is off by at most 24 * 2^-24 * 62 sum |x|.
// A word's eight codes come out as the pairs (0, 4), (1, 5), (2, 6), (3, 7); x is put into the same order.
// The waves of a workgroup take blocks of 128 columns in turn and add their sums through LDS in wave order at the end.
#pragma once

#include "fp8_gemm_common.h"
#include "fp8_quant.h"
#include "rms_norm.h"

namespace dlb {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct W4Args {
  const void* x;
  const uint8_t* q;          // [E][N][K / 2], low nibble = even column
  const void* s;             // [E][N][G] of s_type
  const uint8_t* z;          // [E][N][G] or NULL
  void* y;                   // [rows][N]
  const int32_t* row_start;  // [E] or NULL: one matrix, all rows
  const int32_t* row_end;
  int64_t x_rs, y_rs;
  int64_t q_es, s_es;        // per expert: bytes, scales
  int64_t rows;
  int N, K, G, E;
  int s_type;
};

template <int T>
__device__ __forceinline__ v4f mfma_16x16x32(const v4i& a, const v4i& b, const v4f& c) {
  if (T == kInBf16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

__device__ __forceinline__ float load_scale(const void* s, int type, int64_t i) {
  if (type == kInF32) return static_cast<const float*>(s)[i];
  const uint32_t w = static_cast<const uint16_t*>(s)[i];
  if (type == kInBf16) return __uint_as_float(w << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
}

// Words i of the four quarters of the wave change places with quarters i of the words: quarter q of word i then holds what
// quarter i held in word q.
__device__ __forceinline__ void transpose_quarters(v4i& v) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  const v2u a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const v2u b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const v2u c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const v2u d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v = v4i{static_cast<int>(c[0]), static_cast<int>(c[1]), static_cast<int>(d[0]), static_cast<int>(d[1])};
}

// STEPS = MFMA steps (32 columns) per group: 4, 2, 1 for groups of 128, 64, 32.  A tile is 16 MT rows of x by 16 NT rows of the
// matrix.  Groups below a block of 128 need the 32 columns of a step to be neighbours, so the quarters of the wave exchange words;
// otherwise a quarter keeps its 32 columns and x is read to match.
template <int T, int STEPS, int MT, int NT>
__global__ void __launch_bounds__(512) w4_gemm_kernel(const W4Args p) {
  extern __shared__ float part[];  // [waves][MT][NT][256]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const int quarter = lane >> 4, l16 = lane & 15;
  constexpr bool kTranspose = STEPS < 4;
  constexpr int kGroups = 4 / STEPS;  // of a block
  const uint8_t* wq = p.q;
  int64_t s_base = 0;
  int64_t row0 = static_cast<int64_t>(blockIdx.y) * 16 * MT, row_end = min(p.rows, row0 + 16 * MT);
  if (p.row_start) {
    // the blockIdx.y-th expert that has rows
    int left = blockIdx.y;
    int e = -1;
    for (int e0 = 0; e0 < p.E && e < 0; e0 += 64) {
      const int i = e0 + lane;
      uint64_t some = __ballot(i < p.E && p.row_end[i < p.E ? i : 0] > p.row_start[i < p.E ? i : 0]);
      const int n = __popcll(some);
      if (left >= n) {
        left -= n;
        continue;
      }
      for (; left > 0; --left) some &= some - 1;
      e = e0 + __builtin_ctzll(some);
    }
    if (e < 0) return;
    e = __builtin_amdgcn_readfirstlane(e);
    row0 = max(p.row_start[e], 0), row_end = min(static_cast<int64_t>(p.row_end[e]), p.rows);
    wq += e * p.q_es;
    s_base = e * p.s_es;
  }
  const int blocks = (p.K + 127) / 128;
  const int half = p.K / 2;  // bytes of a row
  int n_row[NT];             // rows past the matrix read its last one and are not stored
#pragma unroll
  for (int n = 0; n < NT; ++n) n_row[n] = min(static_cast<int>(blockIdx.x) * 16 * NT + 16 * n + l16, p.N - 1);
  v4i ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) ones[i] = T == kInBf16 ? 0x3f803f80 : 0x3c003c00;

  for (; row0 < row_end; row0 += 16 * MT) {
    v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
    const char* x_row[MT];
    bool x_on[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int64_t r = row0 + 16 * m + l16;
      x_on[m] = r < row_end;
      x_row[m] = static_cast<const char*>(p.x) + (x_on[m] ? r : row0) * p.x_rs * 2;
    }
    auto load_w = [&](int kb, v4i (&w)[NT]) {
      const int off = kb * 64 + 16 * quarter;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        w[n] = v4i{0, 0, 0, 0};
        if (off < half) w[n] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(wq + static_cast<int64_t>(n_row[n]) * half + off));
      }
    };
    v4i w_now[NT];
    if (wave < blocks) load_w(wave, w_now);
    for (int kb = wave; kb < blocks; kb += waves) {
      v4i w_next[NT];
      if (kb + waves < blocks) load_w(kb + waves, w_next);
      float sc[NT][kGroups], coef[NT][kGroups];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int64_t i = s_base + static_cast<int64_t>(n_row[n]) * p.G + min(kb * kGroups + g, p.G - 1);
          sc[n][g] = load_scale(p.s, p.s_type, i);
          coef[n][g] = -16.f - (p.z ? static_cast<float>(p.z[i]) : 8.f);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (kTranspose) transpose_quarters(w_now[n]);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        v4f sum[MT][NT], xs[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          xs[m] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int n = 0; n < NT; ++n) sum[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int i = g * STEPS; i < (g + 1) * STEPS; ++i) {
          const int k = kb * 128 + (kTranspose ? 32 * i + 8 * quarter : 32 * quarter + 8 * i);
          v4i xf[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            v4i v{0, 0, 0, 0};
            if (x_on[m] && k < p.K) v = *reinterpret_cast<const v4i_el*>(x_row[m] + 2 * k);
            xf[m][0] = __builtin_amdgcn_perm(v[2], v[0], 0x05040100);
            xf[m][1] = __builtin_amdgcn_perm(v[2], v[0], 0x07060302);
            xf[m][2] = __builtin_amdgcn_perm(v[3], v[1], 0x05040100);
            xf[m][3] = __builtin_amdgcn_perm(v[3], v[1], 0x07060302);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) xs[m] = mfma_16x16x32<T>(xf[m], ones, xs[m]);
          constexpr int kBits = T == kInBf16 ? 0x41804180 : 0x4c004c00;
          constexpr int kMask = T == kInBf16 ? 0x00780078 : 0x03c003c0, kUp = T == kInBf16 ? 3 : 6;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int word = w_now[n][i];
            v4i b;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = ((4 * j < kUp ? word << (kUp - 4 * j) : word >> (4 * j - kUp)) & kMask) | kBits;
#pragma unroll
            for (int m = 0; m < MT; ++m) sum[m][n] = mfma_16x16x32<T>(xf[m], b, sum[m][n]);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[m][n][r] = fmaf(sc[n][g], fmaf(coef[n][g], xs[m][r], sum[m][n][r]), acc[m][n][r]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) w_now[n] = w_next[n];
    }
    // lane l holds rows 4 (l / 16) + r, column l % 16 of a tile
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[((wave * MT + m) * NT + n) * 256 + (4 * quarter + r) * 16 + l16] = acc[m][n][r];
    __syncthreads();
    for (int i = tid; i < MT * NT * 256; i += blockDim.x) {
      const int m = i / (NT * 256), n = i / 256 % NT, e = i % 256;
      const int64_t row = row0 + 16 * m + e / 16;
      const int col = static_cast<int>(blockIdx.x) * 16 * NT + 16 * n + e % 16;
      float sum = 0.f;
      for (int w = 0; w < waves; ++w) sum += part[w * MT * NT * 256 + i];
      if (row >= row_end || col >= p.N) continue;
      if (T == kInBf16)
        static_cast<__bf16*>(p.y)[row * p.y_rs + col] = static_cast<__bf16>(sum);
      else
        static_cast<_Float16*>(p.y)[row * p.y_rs + col] = static_cast<_Float16>(sum);
    }
    __syncthreads();
  }
}

// 4-bit quantiser: per group of 32, 64 or 128 columns of a row
//   without zero points  s = max |w| / 7 rounded to its type,             q = clamp(round(w / s) + 8, 0, 15)
//   with them            s = (max(w, 0) - min(w, 0)) / 15 rounded,        z = round(-min(w, 0) / s),  q = clamp(round(w / s) + z, 0, 15)
// A group of zeros has s = 0 and q = 8 (z = 0, q = 0 with zero points).  8 columns a lane, one store of 4 bytes.
struct W4QuantArgs {
  const void* w;
  uint8_t* q;   // [rows][K / 2]
  void* s;      // [rows][G] of the weights' type
  uint8_t* z;   // [rows][G] or NULL
  int64_t rows, w_rs;
  int G, group;
};

template <int T>
__device__ __forceinline__ float round_to_type(float v) {
  if (T == kInBf16) return static_cast<float>(static_cast<__bf16>(v));
  if (T == kInF16) return static_cast<float>(static_cast<_Float16>(v));
  return v;
}

template <int T>
__global__ void __launch_bounds__(256) w4_quant_kernel(const W4QuantArgs p) {
  const int lanes = p.group / 8;  // of a group: 4, 8 or 16
  const int64_t total = p.rows * p.G;
  const int sub = threadIdx.x % lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256 / lanes;
  for (int64_t g = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / lanes; g < total; g += step) {
    const int64_t row = g / p.G, kg = g - row * p.G;
    float v[8];
    quant_unpack8<T>(load_raw8<T>(p.w, row * p.w_rs + kg * p.group + 8 * sub, 8), v);
    float hi = 0.f, lo = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) hi = fmaxf(hi, v[i]), lo = fminf(lo, v[i]);
    for (int off = lanes / 2; off >= 1; off >>= 1) hi = fmaxf(hi, __shfl_xor(hi, off, lanes)), lo = fminf(lo, __shfl_xor(lo, off, lanes));
    const float s = round_to_type<T>(p.z ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f);
    const float zero = p.z ? (s > 0.f ? fminf(rintf(-lo / s), 15.f) : 0.f) : 8.f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = s > 0.f ? fminf(fmaxf(rintf(v[i] / s) + zero, 0.f), 15.f) : zero;
      word |= static_cast<uint32_t>(c) << (4 * i);
    }
    reinterpret_cast<uint32_t*>(p.q)[g * lanes + sub] = word;
    if (sub == 0) {
      if (T == kInF32)
        static_cast<float*>(p.s)[g] = s;
      else if (T == kInBf16)
        static_cast<__bf16*>(p.s)[g] = static_cast<__bf16>(s);
      else
        static_cast<_Float16*>(p.s)[g] = static_cast<_Float16>(s);
      if (p.z) p.z[g] = static_cast<uint8_t>(zero);
    }
  }
}

}  // namespace dlb
