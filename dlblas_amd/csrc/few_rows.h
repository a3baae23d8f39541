// Few 16-bit rows times quantised weights for gfx950, and what is built of it: a product with 4-bit weights and a layer of experts in two kernels.
//
// Bound by the weights' bytes: each goes from memory to a register once, is converted there and meets the rows in v_mfma_f32_16x16x32.  A lane
// holds 32 bytes of one of 16 rows of a matrix, so that a wave reads whole 128-byte lines; which columns a lane's words are is free as long as the
// lanes with the rows take the same.  Weights are
//   e4m3   with one fp32 scale per 128 x 128: exact in 16 bits, sums of 128 columns times the scale in fp32
//   e2m1   with a power of two per 32 columns.  Beside bf16 rows the scale goes into the conversion: e2m1 has two bits of significand and bf16 the
//          range of the scales, so the products stay exact (scales below 2^-124, whose weights are subnormal numbers of bf16, may count as 0).  fp16 has not
//          that range: there the words change places between the quarters of the wave, so that a step is one group, and the group's sum meets its
//          scale in fp32.
// The waves of a workgroup split K and add their sums through LDS in wave order.
#pragma once

#include "mxfp4.h"

namespace dlb {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

enum WeightType : int { kE4m3 = 0, kE2m1 = 1 };

template <int T>
__device__ __forceinline__ v4f mfma_16x16x32(const v4i& a, const v4i& b, const v4f& c) {
  if (T == kInBf16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Words i of the four quarters of the wave change places with quarters i of the words: quarter q of word i then holds what
// quarter i held in word q.
__device__ __forceinline__ void transpose_quarters(v4i& v) {
  const auto a = __builtin_amdgcn_permlane32_swap(static_cast<unsigned>(v[0]), static_cast<unsigned>(v[2]), false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(static_cast<unsigned>(v[1]), static_cast<unsigned>(v[3]), false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v = v4i{static_cast<int>(c[0]), static_cast<int>(c[1]), static_cast<int>(d[0]), static_cast<int>(d[1])};
}
// The value of each quarter in all quarters.
__device__ __forceinline__ void spread_quarters(uint32_t v, uint32_t (&out)[4]) {
  const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const auto lo = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false), hi = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
  out[0] = lo[0], out[1] = lo[1], out[2] = hi[0], out[3] = hi[1];
}

// 2^(s - 127), NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t s) {
  const uint32_t bits = s == 0 ? 0x00400000u : s << 23;
  return __uint_as_float(s == 255 ? 0x7fc00000u : bits);
}

// Eight weights as 16-bit numbers.
template <int T>
__device__ __forceinline__ v4i from_e4m3(int lo, int hi) {
  const unsigned a = static_cast<unsigned>(lo), b = static_cast<unsigned>(hi);
  if (T == kInBf16)
    return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true))};
  return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true)),
             __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true))};
}
template <int T>
__device__ __forceinline__ v4i from_e2m1(int word, float scale) {
  const unsigned w = static_cast<unsigned>(word);
  if (T == kInBf16)
    return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
             __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
}

// A matrix of weights [N][K].  e4m3: q has K bytes a row, s is [ceil(N / 128)][K / 128] fp32; e2m1: K / 2, and [N][K / 32] bytes.
struct Matrix {
  const uint8_t* q;
  const void* s;
  int N, K;
};

// What a wave reads of a matrix: a chunk is 128 bytes of each of 16 rows.
template <int T, int W>
struct Few {
  static constexpr int kCols = W == kE2m1 ? 256 : 128;  // of a chunk
  static constexpr int kSteps = kCols / 32;             // MFMA steps
  static constexpr bool kByGroup = W == kE2m1 && T == kInF16;

  // First column of the eight that quarter q of the rows' lanes takes in step i.
  static __device__ __forceinline__ int column(int q, int i) {
    if (W == kE4m3) return 32 * q + 8 * i;
    return kByGroup ? 64 * (i & 3) + 32 * (i >> 2) + 8 * q : 64 * q + 8 * i;
  }

  struct Weights {
    v4i w[2];
    uint32_t s;  // e2m1: the scales of a lane's two groups; e4m3: the scale's bits
  };

  // 16 rows of a matrix, from row n0 on.
  struct Tile {
    const uint8_t* q;
    const uint8_t* s;
    uint32_t q_bytes, s_bytes;
    __device__ __forceinline__ Tile(const Matrix& m, int n0) {
      const int rows = max(0, min(16, m.N - n0));
      const uint32_t q_pitch = W == kE2m1 ? m.K / 2 : m.K;
      q = m.q + static_cast<int64_t>(n0) * q_pitch, q_bytes = rows * q_pitch;
      if (W == kE2m1)
        s = static_cast<const uint8_t*>(m.s) + static_cast<int64_t>(n0) * (m.K / kMxGroup), s_bytes = rows * (m.K / kMxGroup);
      else
        s = reinterpret_cast<const uint8_t*>(static_cast<const float*>(m.s) + static_cast<int64_t>(n0 / 128) * (m.K / 128)), s_bytes = rows > 0 ? m.K / 32 : 0;
    }
  };

  // Chunk c; `in` (the same for the wave) false: nothing.  Loads are issued either way, none stands behind a branch.
  static __device__ __forceinline__ void load(const Tile& t, int K, int c, bool in, int q, int l16, Weights& o) {
    const uint32_t at = in ? static_cast<uint32_t>(c) * 128 : 0;
    const auto src = make_rsrc(t.q, in ? t.q_bytes : 0);
    if (W == kE4m3) {
#pragma unroll
      for (int i = 0; i < 2; ++i) o.w[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(src, l16 * static_cast<uint32_t>(K) + 32 * q + 16 * i, at, 2));
      o.s = __builtin_amdgcn_raw_buffer_load_b32(make_rsrc(t.s, in ? t.s_bytes : 0), 0, in ? 4 * c : 0, 0);
      return;
    }
    const int G = K / kMxGroup, g = 8 * c + 2 * q;  // the lane's first group of its row
    const auto s_src = make_rsrc(t.s, in ? t.s_bytes : 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool there = g + i < G;  // else it would be the next row's
      o.w[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(src, there ? l16 * static_cast<uint32_t>(K / 2) + 32 * q + 16 * i : kNowhere, at, 2));
    }
    const uint32_t lo = __builtin_amdgcn_raw_buffer_load_b8(s_src, g < G ? l16 * static_cast<uint32_t>(G) + 2 * q : kNowhere, at / 16, 0);
    const uint32_t hi = __builtin_amdgcn_raw_buffer_load_b8(s_src, g + 1 < G ? l16 * static_cast<uint32_t>(G) + 2 * q + 1 : kNowhere, at / 16, 0);
    o.s = lo | hi << 8;
  }

  // acc[m] += rows m times the chunk; lane l receives D[4 (l / 16) + r][l % 16], rows by matrix rows.
  template <int MT>
  static __device__ __forceinline__ void multiply(Weights& w, const v4i (&x)[MT][kSteps], v4f (&acc)[MT]) {
    if (W == kE4m3) {
      v4f sum[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) sum[m] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const v4i f = from_e4m3<T>(w.w[i >> 1][2 * (i & 1)], w.w[i >> 1][2 * (i & 1) + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m) sum[m] = mfma_16x16x32<T>(x[m][i], f, sum[m]);
      }
      const float s = __uint_as_float(w.s);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(s, sum[m][r], acc[m][r]);
      return;
    }
    const float scale[2] = {mx_scale(w.s & 0xffu), mx_scale(w.s >> 8)};
    if (!kByGroup) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const v4i f = from_e2m1<T>(w.w[i >> 2][i & 3], scale[i >> 2]);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = mfma_16x16x32<T>(x[m][i], f, acc[m]);
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t by_group[4];  // of groups 2 i + u
      spread_quarters(__float_as_uint(scale[u]), by_group);
      transpose_quarters(w.w[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v4i f = from_e2m1<T>(w.w[u][i], 1.0f);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const v4f sum = mfma_16x16x32<T>(x[m][4 * u + i], f, v4f{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(__uint_as_float(by_group[i]), sum[r], acc[m][r]);
        }
      }
    }
  }
};

constexpr int kFewWaves = 8;

__device__ __forceinline__ void store1(void* to, int type, int64_t at, float v) {
  if (type == kInBf16)
    static_cast<__bf16*>(to)[at] = static_cast<__bf16>(v);
  else if (type == kInF16)
    static_cast<_Float16*>(to)[at] = static_cast<_Float16>(v);
  else
    static_cast<float*>(to)[at] = v;
}

// Chunks wave, wave + 8, ... of K: the next one is asked for before this one is multiplied.  x_off: of a lane's row m, kNowhere: none.
template <int T, int W, int MT, int NT>
__device__ __forceinline__ void split_k(const typename Few<T, W>::Tile (&tile)[NT], int K, __amdgpu_buffer_rsrc_t x_src, const uint32_t (&x_off)[MT], int wave, int q, int l16,
                                        v4f (&acc)[NT][MT]) {
  typedef Few<T, W> F;
  struct Chunk {
    typename F::Weights w[NT];
    v4i x[MT][F::kSteps];
  };
  const int chunks = (K + F::kCols - 1) / F::kCols;
  auto load = [&](int c, Chunk& k) {
    const bool in = c < chunks;
#pragma unroll
    for (int n = 0; n < NT; ++n) F::load(tile[n], K, c, in, q, l16, k.w[n]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < F::kSteps; ++i) {
        const int col = c * F::kCols + F::column(q, i);
        k.x[m][i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(x_src, x_off[m] != kNowhere && col < K ? x_off[m] + 2 * col : kNowhere, 0, 0));
      }
  };
  auto multiply = [&](Chunk& k) {
#pragma unroll
    for (int n = 0; n < NT; ++n) F::template multiply<MT>(k.w[n], k.x, acc[n]);
  };
  Chunk even, odd;
  load(wave, even);
  for (int c = wave; c < chunks; c += 2 * kFewWaves) {
    load(c + kFewWaves, odd);
    __builtin_amdgcn_sched_barrier(0);
    multiply(even);
    __builtin_amdgcn_sched_barrier(0);
    load(c + 2 * kFewWaves, even);
    __builtin_amdgcn_sched_barrier(0);
    multiply(odd);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ---- one matrix -------------------------------------------------------------------------------------------------------

struct FewArgs {
  const void* x;  // [M][x_rs]
  void* y;        // [M][N]
  int64_t M, x_rs;
  Matrix w;
};

template <int T, int W, int MT, int NT>
__global__ void __launch_bounds__(64 * kFewWaves) few_rows_kernel(const FewArgs p) {
  __shared__ v4f part[kFewWaves][NT * MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int n0 = blockIdx.x * 16 * NT;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 16 * MT;
  const int rows = static_cast<int>(min(p.M - m0, static_cast<int64_t>(16 * MT)));
  const uint32_t pitch = static_cast<uint32_t>(p.x_rs) * 2;
  const auto x_src = make_rsrc(static_cast<const uint8_t*>(p.x) + m0 * p.x_rs * 2, (rows - 1) * pitch + 2 * p.w.K);
  uint32_t x_off[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) x_off[m] = 16 * m + l16 < rows ? (16 * m + l16) * pitch : kNowhere;
  typedef typename Few<T, W>::Tile Tile;
  v4f acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = v4f{0.f, 0.f, 0.f, 0.f};
  if constexpr (NT == 1) {
    const Tile tile[1] = {Tile(p.w, n0)};
    split_k<T, W, MT, 1>(tile, p.w.K, x_src, x_off, wave, q, l16, acc);
  } else {
    const Tile tile[2] = {Tile(p.w, n0), Tile(p.w, n0 + 16)};
    split_k<T, W, MT, 2>(tile, p.w.K, x_src, x_off, wave, q, l16, acc);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) part[wave][n * MT + m][lane] = acc[n][m];
  __syncthreads();
  for (int i = wave; i < NT * MT; i += kFewWaves) {
    v4f sum = part[0][i][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) sum += part[w][i][lane];
    const int n = i / MT, m = i - n * MT, col = n0 + 16 * n + l16;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * m + 4 * q + r;
      if (row < rows && col < p.w.N) store1(p.y, T, (m0 + row) * p.w.N + col, sum[r]);
    }
  }
}

// ---- experts ----------------------------------------------------------------------------------------------------------
//
//   out[t] = sum over the slots j with 0 <= ids[t, j] < E of w[t, j] Down[e] (silu(Gate[e] x[t]) * (Up[e] x[t])),   e = ids[t, j]
//
// The first kernel leaves w silu(g) u of every slot, the second reads it against the experts' second matrices.  No sort in front: there are at most 64
// tokens, a lane of a wave each, so the tokens of an expert are a ballot.  In between the numbers are held as the sum of two bf16, 16 bits of
// significand, which the second kernel's rows take one beside the other: eight tokens and their rests are the 16 rows of an MFMA.  An
// expert that a token names twice counts with the sum of both weights.

constexpr int kFewTokens = 64, kFewTopk = 16, kFewExperts = 1024;

struct ExpertArgs {
  const void* x;         // [T][x_rs]
  const void* ids;       // [T][topk], int32 or int64, through two strides
  const float* weights;  // [T][topk]
  uint16_t* act;         // [2][T topk][I] bf16: the numbers, and what they leave
  void* out;             // [T][H]
  Matrix up, down;       // of expert 0: [2 I][H], [H][I]
  int64_t up_q, up_s, down_q, down_s;  // bytes to the next expert
  int64_t x_rs, ids_s0, ids_s1;
  int T, topk, E, H, I;
  int ids_is64;
};

__device__ __forceinline__ Matrix of_expert(const Matrix& m, int64_t q, int64_t s, int e) {
  return Matrix{m.q + e * q, static_cast<const uint8_t*>(m.s) + e * s, m.N, m.K};
}

__device__ __forceinline__ int expert_of(const ExpertArgs& p, int t, int j) {
  const int64_t at = t * p.ids_s0 + j * p.ids_s1;
  const int64_t e = p.ids_is64 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<const int32_t*>(p.ids)[at];
  return e >= 0 && e < p.E ? static_cast<int>(e) : -1;
}

// Lane i of the result: the lane of the i-th bit of the mask.
__device__ __forceinline__ int nth_lane(uint64_t mask, int lane) {
  const uint64_t below = (uint64_t{1} << lane) - 1;
  const bool mine = mask >> lane & 1;
  const int to = mine ? __popcll(mask & below) : __popcll(mask) + __popcll(~mask & below);
  return __builtin_amdgcn_ds_permute(to * 4, lane);
}

// silu(g) u
__device__ __forceinline__ float gated(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

// A workgroup takes 16 rows of Gate and the same of Up, of expert blockIdx.y, or where there are more experts than slots of that slot's expert, if
// it is the first to name it.
template <int T, int W, int MT>
__global__ void __launch_bounds__(64 * kFewWaves) experts_up_kernel(const ExpertArgs p) {
  __shared__ v4f part[kFewWaves][2 * MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int slots = p.T * p.topk, y = blockIdx.y;
  const bool by_slot = p.E > slots;
  const int e = __builtin_amdgcn_readfirstlane(by_slot ? expert_of(p, y / p.topk, y % p.topk) : y);
  if (e < 0) return;
  int first = -1;  // the slot of this lane's token
  float weight = 0.f;
  const int token = min(lane, p.T - 1);
  for (int j0 = 0; j0 < p.topk; j0 += 8) {  // eight at a time on their way
    int named[8];
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = min(j0 + i, p.topk - 1);
      named[i] = expert_of(p, token, j), w[i] = p.weights[token * p.topk + j];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (lane >= p.T || j0 + i >= p.topk || named[i] != e) continue;
      if (first < 0) first = token * p.topk + j0 + i;
      weight += w[i];
    }
  }
  const uint64_t mask = __ballot(first >= 0);
  if (mask == 0) return;
  if (by_slot && __shfl(first, __builtin_ctzll(mask)) != y) return;
  const int rows = __popcll(mask), token_of = nth_lane(mask, lane);
  typedef typename Few<T, W>::Tile Tile;
  const Matrix up = of_expert(p.up, p.up_q, p.up_s, e);
  const int n0 = blockIdx.x * 16;
  const Tile tile[2] = {Tile(up, n0), Tile(up, p.I + n0)};
  const auto x_src = make_rsrc(p.x, static_cast<uint32_t>((p.T - 1) * p.x_rs + p.H) * 2);
  const int64_t rest = static_cast<int64_t>(slots) * p.I;
  for (int b = 0; b < rows; b += 16 * MT) {
    uint32_t x_off[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int i = b + 16 * m + l16;
      const int token = __shfl(token_of, i & 63);
      x_off[m] = i < rows ? static_cast<uint32_t>(token * p.x_rs) * 2 : kNowhere;
    }
    v4f acc[2][MT];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[n][m] = v4f{0.f, 0.f, 0.f, 0.f};
    split_k<T, W, MT, 2>(tile, p.H, x_src, x_off, wave, q, l16, acc);
    if (b > 0) __syncthreads();
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) part[wave][n * MT + m][lane] = acc[n][m];
    __syncthreads();
    if (wave >= MT) continue;
    v4f g = part[0][wave][lane], u = part[0][MT + wave][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) g += part[w][wave][lane], u += part[w][MT + wave][lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = b + 16 * wave + 4 * q + r;
      const int token = __shfl(token_of, i & 63);
      const int slot = __shfl(first, token);
      const float v = gated(g[r], u[r]) * __shfl(weight, token);
      if (i >= rows) continue;
      const __bf16 hi = static_cast<__bf16>(v);
      const float f = static_cast<float>(hi);
      const __bf16 lo = static_cast<__bf16>(fabsf(f) == __builtin_inff() ? 0.f : v - f);
      uint16_t* const to = p.act + static_cast<int64_t>(slot) * p.I + n0 + l16;
      to[0] = __builtin_bit_cast(uint16_t, hi), to[rest] = __builtin_bit_cast(uint16_t, lo);
    }
  }
}

// A workgroup takes 16 columns of the output of all tokens.  Its work is a list of experts, several times where one has more than 8 MT tokens, by chunks
// of their K = I; each wave takes a run of that and adds its sums up in an LDS table of its own, and the tables are added in wave order.
template <int TO, int W, int MT>
__global__ void __launch_bounds__(64 * kFewWaves) experts_down_kernel(const ExpertArgs p) {
  typedef Few<kInBf16, W> F;
  extern __shared__ __attribute__((aligned(16))) char dynamic[];  // [waves][T][16] sums
  __shared__ int count[kFewExperts];
  __shared__ int16_t ids[kFewTopk][kFewTokens];
  __shared__ int32_t entry[kFewTokens * kFewTopk];  // expert, pass << 16
  __shared__ int entries;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int slots = p.T * p.topk;
  constexpr int kThreads = 64 * kFewWaves;
  for (int i = tid; i < p.E; i += kThreads) count[i] = 0;
  float* const sums = reinterpret_cast<float*>(dynamic) + wave * p.T * 16;
  for (int i = lane; i < p.T * 16; i += 64) sums[i] = 0.f;
  __syncthreads();
  for (int s = tid; s < slots; s += kThreads) {
    const int t = s / p.topk, j = s - t * p.topk, e = expert_of(p, t, j);
    ids[j][t] = static_cast<int16_t>(e);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  if (wave == 0) {
    // a token that names an expert twice counts twice here: at most an entry without rows
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
      const int passes = e0 + lane < p.E ? (count[e0 + lane] + 8 * MT - 1) / (8 * MT) : 0;
      int upto = passes;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(upto, off);
        if (lane >= off) upto += v;
      }
      for (int i = 0; i < passes; ++i) entry[before + upto - passes + i] = (e0 + lane) | i << 16;
      before += __shfl(upto, 63);
    }
    if (lane == 0) entries = before;
  }
  __syncthreads();
  const int n0 = blockIdx.x * 16;
  const int chunks = (p.I + F::kCols - 1) / F::kCols;
  const int total = __builtin_amdgcn_readfirstlane(entries) * chunks;
  const int each = (total + kFewWaves - 1) / kFewWaves;
  const int start = min(total, wave * each), end = min(total, start + each);
  const uint32_t rest = static_cast<uint32_t>(slots) * p.I * 2;
  const auto x_src = make_rsrc(p.act, 2 * rest);

  struct Chunk {
    typename F::Weights w[1];
    v4i x[MT][F::kSteps];
  };
  v4f acc[1][MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[0][m] = v4f{0.f, 0.f, 0.f, 0.f};
  // the rows of the entry whose chunks are being asked for
  uint32_t x_off[MT];
  const uint8_t *w_q = p.down.q, *w_s = static_cast<const uint8_t*>(p.down.s);
  auto tokens_of = [&](int en, int& slot_of) {  // the lane's token's slot; the tokens' mask
    const int e = en & 0xffff;
    slot_of = -1;
    for (int j = p.topk - 1; j >= 0; --j)
      if (lane < p.T && ids[j][lane] == e) slot_of = lane * p.topk + j;
    return __ballot(slot_of >= 0);
  };
  auto point_at = [&](int i) {
    const int en = __builtin_amdgcn_readfirstlane(entry[i]);
    int slot_of;
    const uint64_t mask = tokens_of(en, slot_of);
    const int rows = __popcll(mask), token_of = nth_lane(mask, lane), first = (en >> 16) * 8 * MT;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = first + 8 * m + (l16 & 7);
      const int slot = __shfl(slot_of, __shfl(token_of, r & 63));
      x_off[m] = r < rows ? static_cast<uint32_t>(slot) * p.I * 2 + (l16 >> 3) * rest : kNowhere;
    }
    w_q = p.down.q + (en & 0xffff) * p.down_q, w_s = static_cast<const uint8_t*>(p.down.s) + (en & 0xffff) * p.down_s;
  };
  int l_entry = start / max(chunks, 1), l_chunk = start - l_entry * chunks, l_left = end - start;
  if (l_left > 0) point_at(l_entry);
  auto load_next = [&](Chunk& k) {
    const bool in = l_left > 0;
    const typename F::Tile tile(Matrix{w_q, w_s, p.H, p.I}, n0);
    F::load(tile, p.I, l_chunk, in, q, l16, k.w[0]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < F::kSteps; ++i) {
        const int col = l_chunk * F::kCols + F::column(q, i);
        k.x[m][i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(x_src, in && x_off[m] != kNowhere && col < p.I ? x_off[m] + 2 * col : kNowhere, 0, 0));
      }
    if (--l_left > 0 && ++l_chunk == chunks) l_chunk = 0, point_at(++l_entry);
  };
  int m_entry = l_entry, m_chunk = l_chunk, m_left = l_left;
  // the sums of an entry's rows go to their tokens
  auto leave = [&](int i) {
    const int en = __builtin_amdgcn_readfirstlane(entry[i]);
    int slot_of;
    const uint64_t mask = tokens_of(en, slot_of);
    const int rows = __popcll(mask), token_of = nth_lane(mask, lane), first = (en >> 16) * 8 * MT;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = acc[0][m][r] + __shfl_xor(acc[0][m][r], 32);  // a token's numbers and what they left
        const int i = first + 8 * m + (4 * q + r & 7);
        const int token = __shfl(token_of, i & 63);
        if (q < 2 && i < rows) sums[token * 16 + l16] += v;
        acc[0][m][r] = 0.f;
      }
  };
  auto multiply = [&](Chunk& k) {
    F::template multiply<MT>(k.w[0], k.x, acc[0]);
    if (m_left > 0 && (--m_left == 0 || ++m_chunk == chunks)) {
      leave(m_entry);
      m_chunk = 0, ++m_entry;
    }
  };
  if (start < end) {
    Chunk even, odd;
    load_next(even);
    for (int i = start; i < end; i += 2) {
      load_next(odd);
      __builtin_amdgcn_sched_barrier(0);
      multiply(even);
      __builtin_amdgcn_sched_barrier(0);
      load_next(even);
      __builtin_amdgcn_sched_barrier(0);
      multiply(odd);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __syncthreads();
  const float* const all = reinterpret_cast<const float*>(dynamic);
  for (int i = tid; i < p.T * 16; i += kThreads) {
    float v = all[i];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) v += all[w * p.T * 16 + i];
    const int t = i >> 4, col = n0 + (i & 15);
    if (col < p.H) store1(p.out, TO, static_cast<int64_t>(t) * p.H + col, v);
  }
}

}  // namespace dlb
