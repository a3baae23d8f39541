// Few 16-bit rows times quantised weights for gfx950, and what is built of it: a product with 4-bit weights and a layer of experts in two kernels.
//
// Bound by the weights' bytes: each comes from memory once, is converted in registers and meets the rows in v_mfma_f32_16x16x32.  Weights are
//   e4m3   with one fp32 scale per 128 x 128: exact in 16 bits, sums of 128 columns times the scale in fp32
//   e2m1   with a power of two per 32 columns.  Beside bf16 rows the scale goes into the conversion: e2m1 has two bits of significand and bf16 the
//          range of the scales but for their ends, so the products stay exact.  A chunk with a scale at one of those scales its groups' sums in fp32, by what
//          the conversion does not take.  fp16 has not that range: there a group's sum always meets its scale in fp32.
// Waves split K and add their sums through LDS in wave order.
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

// What is the same for the lanes of a wave, in scalar registers: a buffer that the compiler cannot see to be that costs a loop over the lanes a load.
__device__ __forceinline__ uint32_t in_scalar(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const uint8_t* in_scalar(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint64_t lo = in_scalar(static_cast<uint32_t>(v)), hi = in_scalar(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const uint8_t*>(hi << 32 | lo);
}

// A matrix of weights [N][K].  e4m3: q has K bytes a row, s is [ceil(N / 128)][K / 128] fp32; e2m1: K / 2, and [N][K / 32] bytes.
struct Matrix {
  const uint8_t* q;
  const void* s;
  int N, K;
};

// A wave's own stream: chunks of 128 bytes of each row of NT tiles of 16 weight rows, and of R rows of x, come into a ring of DEPTH chunks in LDS that
// no other wave reads, so nothing but the wave's own counter of loads is waited for.  They go through LDS because of the order of the lanes: an MFMA
// wants neighbouring rows in neighbouring lanes, and loaded that way every lane touches a cache line of its own, 64 a load, which held 32 experts x 4
// rows x 4096 x 7168 e4m3 at 250 us however much was on its way.  Here eight lanes share a line, and all of it is asked for at once: chunks of half a line
// of e2m1 150 us, and the products themselves cost nothing of that.
//
// Rows of x are 16-bit numbers, or with F32 fp32 ones, R / 2 of them: each is the sum of three bf16, the nearest, the nearest to what that leaves, and the rest, which
// has six bits at most (parts below 2^-126 may count as 0).  Every part has a product of its own.  A lane makes the parts of eight numbers, those of one step in R / 2 rows of
// the MFMA and of the next in the R / 2 behind them, so that none makes what another has; a product of one step then fills those rows, and what it leaves in the others is
// of no use.  Instructions bound this (16 tokens x 8 of 32 experts, 7168 x 2048 e2m1, eight tokens a pass: 102 us, with lanes that exchange their parts, first and second in the
// rows of one product, 103; rows of 16 bits 73).  Sums of the first parts stay apart: what an infinity leaves is no number.
//
// A 16-byte piece of a row lies at another place of it, by the row, so that a read of 16 rows meets every bank once: of x piece ^ row, of weights
// piece ^ (row / 2).  Steps of an MFMA are 32 columns: of e4m3 eight from each quarter's 16-byte piece, of e2m1 a group, a word of its 16 bytes a
// quarter.  The eight scales of a row's chunk of e2m1 start at any byte: they come as the two or three words they lie in.
constexpr int stream_columns(int weights) { return weights == kE4m3 ? 128 : 256; }
constexpr int kStreamTile = 2048 + 256;  // bytes of a tile's chunk: codes, and behind them scales
constexpr int stream_x_loads(int weights, int R) { return R * stream_columns(weights) / 512; }
constexpr int stream_bytes(int weights, int R, int NT) { return NT * kStreamTile + R * stream_columns(weights) * 2; }
// Chunks of a ring of `waves` waves in `bytes` of LDS.
constexpr int stream_depth(int weights, int R, int NT, int waves, int bytes) {
  const int depth = bytes / (waves * stream_bytes(weights, R, NT));
  return depth > 6 ? 6 : depth;
}

template <int T, int W, int R, int NT, int DEPTH, bool F32 = false>
struct Stream {
  static constexpr int kCols = stream_columns(W), kSteps = kCols / 32, kXRows = F32 ? R / 2 : R, kXSize = F32 ? 4 : 2;
  static constexpr int kXPitch = kXSize * kCols, kXLoads = stream_x_loads(W, R), kXLanes = kXPitch / 16;  // lanes of a load that share a row of x
  static constexpr int kChunk = stream_bytes(W, R, NT), kBytes = DEPTH * kChunk;
  static constexpr int kLoads = NT * 3 + kXLoads;  // of a chunk
  static_assert((R == 4 || R == 8 || R == 16) && DEPTH >= 2 && (DEPTH - 1) * kLoads < 64, "whole loads of x, a counter of six bits");
  static_assert(!F32 || T == kInBf16, "parts of fp32");

  // 16 rows of a matrix, from row n0 on; past its end the last that it has (a buffer of no bytes would not do: its end is compared with what a chunk's offset leaves of it).
  struct Tile {
    const uint8_t *q, *s;
    uint32_t q_bytes, s_bytes;
    __device__ __forceinline__ void point_at(const Matrix& m, int n0) {
      n0 = min(n0, (m.N - 1) / 16 * 16);
      const int rows = min(16, m.N - n0);
      const uint32_t q_pitch = W == kE2m1 ? m.K / 2 : m.K;
      q = m.q + static_cast<int64_t>(n0) * q_pitch, q_bytes = rows * q_pitch;
      if (W == kE2m1) {  // 16 rows of scales are whole words, so every tile starts as far into one as the matrix does
        const uint32_t into = reinterpret_cast<uintptr_t>(m.s) & 3;
        s = static_cast<const uint8_t*>(m.s) - into + static_cast<int64_t>(n0) * (m.K / kMxGroup), s_bytes = (into + rows * (m.K / kMxGroup) + 3) & ~3u;
      } else {
        s = reinterpret_cast<const uint8_t*>(static_cast<const float*>(m.s) + static_cast<int64_t>(n0 / 128) * (m.K / 128)), s_bytes = m.K / 32;
      }
      q = in_scalar(q), s = in_scalar(s), q_bytes = in_scalar(q_bytes), s_bytes = in_scalar(s_bytes);
    }
  };

  const uint8_t* ring;  // this wave's
  mx_lds_bytes ring_to;
  int K, chunks, row_bytes;
  const uint8_t* x;
  uint32_t x_bytes;
  uint32_t w_at, s_at;  // where a lane starts in a tile, and in its scales
  int w_from, x_from, s_from;   // where it reads in a chunk
  int q, l16;
  uint32_t x_at[kXLoads];  // its row of x of each load with its piece; past the end of every buffer: none
  Tile tile[NT];
  v4f acc[NT];
  // With F32, of the steps g + kTurns i: rows kXRows g to kXRows (g + 1) - 1, the others are of no use.
  static constexpr int kTurns = F32 && W == kE2m1 && R <= 8 ? 4 : 2;
  struct Sums {
    v4f first[kTurns], rest[kTurns];  // of the first parts, of the others
    __device__ __forceinline__ void clear() {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) first[i] = rest[i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
  };
  Sums sums[F32 ? NT : 1];

  __device__ __forceinline__ Stream(uint8_t* lds, int wave, int lane, int columns, const void* x_base, uint32_t bytes, const void* scales)
      : ring(lds + wave * kBytes), ring_to((mx_lds_bytes)lds + wave * kBytes), K(columns), chunks((columns + kCols - 1) / kCols), row_bytes(W == kE4m3 ? columns : columns / 2),
        x(in_scalar(static_cast<const uint8_t*>(x_base))), x_bytes(in_scalar(bytes)), q(lane >> 4), l16(lane & 15) {
    const int row = lane >> 3, x_row16 = l16 & (kXRows - 1);
    w_at = row * row_bytes + ((lane & 7) ^ (row >> 1)) * 16;
    w_from = l16 * 128 + (W == kE4m3 ? ((q ^ (l16 >> 1)) & 7) * 16 : (l16 >> 1) * 16 + 4 * q);
    // of fp32 two pieces, in lanes of the next rows those of the step behind
    const int second = F32 ? (l16 / kXRows & (kTurns - 1)) * (W == kE4m3 ? 2 : 8) : 0;
    x_from = x_row16 * kXPitch + (((W == kE4m3 ? 2 * q : q) * (F32 ? 2 : 1) + second) ^ x_swizzle(x_row16)) * 16;
    const uint32_t into = reinterpret_cast<uintptr_t>(scales) & 3, pitch = columns / kMxGroup;
    const int lanes = (into | pitch % 4) == 0 ? 1 : 2;  // log2 of those of a row: of whole words two, otherwise three of four
    const uint32_t row_of = lane >> lanes, word = lane & ((1 << lanes) - 1);
    s_at = W == kE4m3 ? 0 : row_of < 16 && word < 3 ? ((into + row_of * pitch) & ~3u) + 4 * word : kNowhere;
    s_from = W == kE4m3 ? 2048 : 2048 + (l16 << (lanes + 2)) + ((into + l16 * pitch) & 3) + 2 * q;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = v4f{0.f, 0.f, 0.f, 0.f}, sums[F32 ? n : 0].clear();
  }
  // A row's 16-byte piece c of x lies at c ^ this.  Of fp32 a turn of 16 lanes holds every row with two quarters, whose pieces differ in bit 1 (e2m1) or 2 (e4m3), and half of
  // the rows have a step, which is bit 3 (e2m1) or 1 (e4m3), behind the others: the rows take the other three bits.
  static __device__ __forceinline__ int x_swizzle(int row) { return !F32 ? row : W == kE4m3 ? (row & 3) | (row & 4) << 1 : (row & 1) | (row & 6) << 1; }
  // Row of x that load j brings for a lane, and the lane's column there.
  static __device__ __forceinline__ int x_row(int lane, int j) { return 64 / kXLanes * j + lane / kXLanes; }
  static __device__ __forceinline__ int x_column(int lane, int j) { return (lane % kXLanes ^ x_swizzle(x_row(lane, j) & 15)) * (16 / kXSize); }
  // at: byte of that row, kNowhere: none
  __device__ __forceinline__ void set_row(int lane, int j, uint32_t at) { x_at[j] = at == kNowhere ? kNowhere : at + kXSize * x_column(lane, j); }

  // Chunk c into place d; `in` false (the same for the wave): nothing is brought.  Loads are issued either way.
  __device__ __forceinline__ void load(int d, int lane, int c, bool in) {
    const mx_lds_bytes to = ring_to + d * kChunk;
    const uint32_t at = in ? static_cast<uint32_t>(c) * 128 : 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // Past the end of a row of e2m1 a lane brings the next one's codes, which meet zeros of x.
      const auto src = make_rsrc(tile[n].q, in ? tile[n].q_bytes : 0);
      load_to_lds<2>(src, to + n * kStreamTile, w_at, at);
      // eight rows further on row / 2 has another third bit: the other half of the chunk
      const uint32_t half = ((lane & 7) ^ (lane >> 4)) < 4 ? 64u : -64u;
      load_to_lds<2>(src, to + n * kStreamTile + 1024, w_at + half + 8 * row_bytes, at);
      load4_to_lds(make_rsrc(tile[n].s, in ? tile[n].s_bytes : 0), to + n * kStreamTile + 2048, s_at, in ? (W == kE4m3 ? 4 : 8) * c : 0);
    }
#pragma unroll
    for (int j = 0; j < kXLoads; ++j) {
      const bool there = W == kE4m3 || c * kCols + x_column(lane, j) < K;
      load_to_lds<0>(make_rsrc(x, in ? x_bytes : 0), to + NT * kStreamTile + j * 1024, there ? x_at[j] : kNowhere, in ? static_cast<uint32_t>(c) * kXPitch : 0);
    }
  }

  // Eight fp32 numbers as three parts each.
  static __device__ __forceinline__ void parts(const v4f (&v)[2], v4i (&part)[3]) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    typedef float v2f __attribute__((ext_vector_type(2)));
    // -1 beside 0, out of the compiler's sight: it would write the lower one as the constant -1.0 of the instruction, which is that of fp32, the upper one
    uint32_t lower = 0xbf80u, upper = 0xbf800000u;
    asm("" : "+s"(lower), "+s"(upper));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v2f f{v[i / 2][2 * (i & 1)], v[i / 2][2 * (i & 1) + 1]};
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const v2bf b = __builtin_convertvector(f, v2bf);
        part[k][i] = __builtin_bit_cast(int, b);
        f = v2f{__builtin_amdgcn_fdot2_f32_bf16(b, __builtin_bit_cast(v2bf, lower), f[0], false), __builtin_amdgcn_fdot2_f32_bf16(b, __builtin_bit_cast(v2bf, upper), f[1], false)};
      }
    }
  }

  // The scales of e2m1 of row l16 of every tile, of groups 2 q and 2 q + 1 of a chunk; zeros past the end of the row.  Beside bf16: whether there is a weight, in any row of the wave,
  // that it does not hold.  The first test takes three scales more than the ends, 253 to 255 and 0 to 4 by five bits; a group of zeros, whose scale is 0, passes the second
  // (64 x 7168 x 18432 with a group of zeros in 63: 76 us, without it 98; with none 58).
  __device__ __forceinline__ bool scales(const uint8_t* from, uint32_t scaled, uint32_t (&two)[NT]) const {
    bool beyond = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint32_t of = *reinterpret_cast<const mx_two_bytes*>(from + n * kStreamTile + s_from);
      two[n] = of & scaled;
      const uint32_t behind = ((of & scaled) | (0x8080u & ~scaled)) + 0x0303u;  // a carry is one of a byte that is beyond
      beyond |= (behind & 0xf8u) == 0 || (behind & 0xf800u) == 0;
    }
    if (T != kInBf16 || __builtin_amdgcn_ballot_w64(beyond) == 0) return false;
    bool out = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t s = two[n] >> 8 * u & 0xff, in_row = scaled >> 8 * u & 0xff;
        const v4i w = *reinterpret_cast<const v4i*>(from + n * kStreamTile + l16 * 128 + ((2 * q + u) ^ (l16 >> 1)) * 16);
        out |= in_row && (s >= 253 || (s < 2 && ((w[0] | w[1] | w[2] | w[3]) & 0x77777777) != 0));
      }
    return __builtin_amdgcn_ballot_w64(out) != 0;
  }
  // Those of groups 2 i + u for all quarters, each of which has two: as fp32, for bf16 by the exponent alone.
  static __device__ __forceinline__ void spread(uint32_t two, uint32_t (&by_group)[2][4]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) spread_quarters(T == kInBf16 ? (two >> 8 * u & 0xff) << 23 : __float_as_uint(mx_scale(two >> 8 * u & 0xff)), by_group[u]);
  }
  // A scale as one that bf16 has for every code, 2^-125 ... 2^125, and the rest of it, for sums in fp32: 2^-2 ... 2^2, NaN of NaN.
  static __device__ __forceinline__ void part_scale(uint32_t scale, float& inner, float& outer) {
    const uint32_t s = scale >> 23, near = min(max(s, 2u), 252u);
    inner = __uint_as_float(near << 23), outer = __uint_as_float(s == 255 ? 0x7fc00000u : (127 + s - near) << 23);
  }

  __device__ __forceinline__ void multiply_rows(const uint8_t* from, uint32_t scaled) {
    if constexpr (W == kE4m3)
      multiply_rows_e4m3(from);
    else if (uint32_t two[NT]; scales(from, scaled, two))
      multiply_rows_e2m1<T == kInBf16>(from, two);
    else
      multiply_rows_e2m1<false>(from, two);
  }
  __device__ __forceinline__ void multiply_rows_e4m3(const uint8_t* from) {
    v4i xf[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) xf[i] = *reinterpret_cast<const v4i*>(from + NT * kStreamTile + (x_from ^ (128 * (i >> 1) + 16 * (i & 1))));
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* const codes = from + n * kStreamTile;
      v4f sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const v4i v = *reinterpret_cast<const v4i*>(codes + (w_from ^ 64 * u));
#pragma unroll
        for (int i = 0; i < 2; ++i) sum = mfma_16x16x32<T>(xf[2 * u + i], from_e4m3<T>(v[2 * i], v[2 * i + 1]), sum);
      }
      const float s = *reinterpret_cast<const float*>(codes + s_from);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[n][r] = fmaf(s, sum[r], acc[n][r]);
    }
  }
  template <bool BEYOND>
  __device__ __forceinline__ void multiply_rows_e2m1(const uint8_t* from, const uint32_t (&two)[NT]) {
    v4i xf[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) xf[i] = *reinterpret_cast<const v4i*>(from + NT * kStreamTile + (x_from ^ 64 * i));
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* const codes = from + n * kStreamTile;
      uint32_t by_group[2][4];
      spread(two[n], by_group);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const uint32_t scale = by_group[i & 1][i >> 1 & 3];
        float inner = T == kInBf16 ? __uint_as_float(scale) : 1.0f, outer = __uint_as_float(scale);
        if (BEYOND) part_scale(scale, inner, outer);
        const v4i f = from_e2m1<T>(*reinterpret_cast<const int*>(codes + (w_from ^ 16 * i)), inner);
        if (T == kInBf16 && !BEYOND) {
          acc[n] = mfma_16x16x32<T>(xf[i], f, acc[n]);
          continue;
        }
        const v4f sum = mfma_16x16x32<T>(xf[i], f, v4f{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[n][r] = fmaf(outer, sum[r], acc[n][r]);
        __builtin_amdgcn_sched_barrier(0);  // the sums of all steps would not fit the registers
      }
    }
  }

  // The same for rows of fp32.
  __device__ __forceinline__ void multiply_parts(const uint8_t* from, uint32_t scaled) {
    if constexpr (W == kE4m3)
      multiply_parts_e4m3(from);
    else if (uint32_t two[NT]; scales(from, scaled, two))
      multiply_parts_e2m1<true>(from, two);
    else
      multiply_parts_e2m1<false>(from, two);
  }
  __device__ __forceinline__ void load_raw(const uint8_t* from, v4f (&raw)[kSteps / kTurns][2]) const {
#pragma unroll
    for (int i = 0; i < kSteps / kTurns; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) raw[i][h] = *reinterpret_cast<const v4f*>(from + NT * kStreamTile + (x_from ^ (128 * kTurns * i + 16 * h)));
  }
  // sums + the parts times a fragment
  static __device__ __forceinline__ void add_product(const v4i (&part)[3], const v4i& f, v4f& first, v4f& rest) {
    first = mfma_16x16x32<T>(part[0], f, first);
    rest = mfma_16x16x32<T>(part[2], f, mfma_16x16x32<T>(part[1], f, rest));
  }
  __device__ __forceinline__ void multiply_parts_e4m3(const uint8_t* from) {
    v4f raw[kSteps / kTurns][2];
    load_raw(from, raw);
    v4i codes[NT][2];
    Sums sum[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int u = 0; u < 2; ++u) codes[n][u] = *reinterpret_cast<const v4i*>(from + n * kStreamTile + (w_from ^ 64 * u));
      sum[n].clear();
    }
    v4i part[3];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i % kTurns == 0) parts(raw[i / kTurns], part);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        add_product(part, from_e4m3<T>(codes[n][i >> 1][2 * (i & 1)], codes[n][i >> 1][2 * (i & 1) + 1]), sum[n].first[i % kTurns], sum[n].rest[i % kTurns]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float s = *reinterpret_cast<const float*>(from + n * kStreamTile + s_from);
#pragma unroll
      for (int i = 0; i < kTurns; ++i) add_scaled(sums[n], i, s, sum[n].first[i], sum[n].rest[i]);
    }
  }
  static __device__ __forceinline__ void add_scaled(Sums& to, int turn, float s, const v4f& first, const v4f& rest) {
#pragma unroll
    for (int r = 0; r < 4; ++r) to.first[turn][r] = fmaf(s, first[r], to.first[turn][r]), to.rest[turn][r] = fmaf(s, rest[r], to.rest[turn][r]);
  }
  template <bool BEYOND>
  __device__ __forceinline__ void multiply_parts_e2m1(const uint8_t* from, const uint32_t (&two)[NT]) {
    v4f raw[kSteps / kTurns][2];
    load_raw(from, raw);
    int codes[NT][kSteps];
    uint32_t by_group[NT][2][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) codes[n][i] = *reinterpret_cast<const int*>(from + n * kStreamTile + (w_from ^ 16 * i));
      spread(two[n], by_group[n]);
    }
    v4i part[3];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int turn = i % kTurns;
      if (turn == 0) parts(raw[i / kTurns], part);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t scale = by_group[n][i & 1][i >> 1 & 3];
        if (!BEYOND) {
          add_product(part, from_e2m1<T>(codes[n][i], __uint_as_float(scale)), sums[n].first[turn], sums[n].rest[turn]);
          continue;
        }
        float inner, outer;
        part_scale(scale, inner, outer);
        v4f first{0.f, 0.f, 0.f, 0.f}, rest{0.f, 0.f, 0.f, 0.f};
        add_product(part, from_e2m1<T>(codes[n][i], inner), first, rest);
        add_scaled(sums[n], turn, outer, first, rest);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // Chunk c, in place d and behind it DEPTH - 1 others, times its rows: lane l of acc[n] has rows 4 (l / 16) + r, column l % 16, with F32 sums[n].
  __device__ __forceinline__ void multiply(int d, int c) {
    const uint32_t scaled = mx_scales_in_row(K / kMxGroup - 8 * c - 2 * q);
    wait_loads<(DEPTH - 1) * kLoads>();  // in order
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t* const from = ring + d * kChunk;  // what is ^ed is within what a row has of a chunk
    if constexpr (F32)
      multiply_parts(from, scaled);
    else
      multiply_rows(from, scaled);
    // what is read of this place has arrived before its next chunk is asked for
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }

  // Chunks wave, wave + waves, ... of K.
  __device__ __forceinline__ void split_k(int lane, int wave, int waves) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      load(d, lane, wave + d * waves, wave + d * waves < chunks);
      __builtin_amdgcn_sched_barrier(0);
    }
    for (int c = wave; c < chunks; c += DEPTH * waves) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        multiply(d, c + d * waves);
        const int next = c + (DEPTH + d) * waves;
        load(d, lane, next, next < chunks);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    wait_loads<0>();  // nothing is on its way into LDS any more
  }
};

__device__ __forceinline__ void store1(void* to, int type, int64_t at, float v) {
  if (type == kInBf16)
    static_cast<__bf16*>(to)[at] = static_cast<__bf16>(v);
  else
    static_cast<_Float16*>(to)[at] = static_cast<_Float16>(v);
}

// ---- one matrix -------------------------------------------------------------------------------------------------------

struct FewArgs {
  const void* x;  // [M][x_rs]
  void* y;        // [M][N]
  int64_t M, x_rs;
  Matrix w;
};

template <int W, int R, int NT>
struct FewShape {
  static constexpr int kBudget = 156 * 1024, kWaves = 8 * 2 * stream_bytes(W, R, NT) <= kBudget ? 8 : 4, kDepth = stream_depth(W, R, NT, kWaves, kBudget);
  static constexpr int kLds = kWaves * kDepth * stream_bytes(W, R, NT);
  static_assert(kLds >= kWaves * NT * 1024, "room for the waves' sums");
};

// R rows of x against 16 NT rows of the matrix.  blockIdx.y: eight column tiles, one for each XCD, blockIdx.x: those tiles by the blocks of R rows, so that the
// workgroups that share weights run beside each other on one XCD.
template <int T, int W, int R, int NT>
__global__ void __launch_bounds__(64 * (FewShape<W, R, NT>::kWaves)) few_rows_kernel(const FewArgs p) {
  typedef FewShape<W, R, NT> Shape;
  typedef Stream<T, W, R, NT, Shape::kDepth> S;
  constexpr int kWaves = Shape::kWaves;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int n0 = (blockIdx.y * 8 + blockIdx.x % 8) * 16 * NT;
  if (n0 >= p.w.N) return;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x / 8) * R;
  const int rows = static_cast<int>(min(p.M - m0, static_cast<int64_t>(R)));
  const uint32_t pitch = static_cast<uint32_t>(p.x_rs) * 2;
  S s(lds, wave, lane, p.w.K, static_cast<const uint8_t*>(p.x) + m0 * p.x_rs * 2, (rows - 1) * pitch + 2 * p.w.K, p.w.s);
#pragma unroll
  for (int n = 0; n < NT; ++n) s.tile[n].point_at(p.w, n0 + 16 * n);
#pragma unroll
  for (int j = 0; j < S::kXLoads; ++j) s.set_row(lane, j, S::x_row(lane, j) < rows ? S::x_row(lane, j) * pitch : kNowhere);
  s.split_k(lane, wave, kWaves);
  __syncthreads();
  v4f* const part = reinterpret_cast<v4f*>(lds);  // [waves][NT][64]
#pragma unroll
  for (int n = 0; n < NT; ++n) part[(wave * NT + n) * 64 + lane] = s.acc[n];
  __syncthreads();
  if (wave >= NT) return;
  v4f sum = part[wave * 64 + lane];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += part[(w * NT + wave) * 64 + lane];
  const int col = n0 + 16 * wave + l16;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = 4 * q + r;
    if (row < rows && col < p.w.N) store1(p.y, T, (m0 + row) * p.w.N + col, sum[r]);
  }
}

// ---- experts ----------------------------------------------------------------------------------------------------------
//
//   out[t] = sum over the slots j with 0 <= ids[t, j] < E of w[t, j] Down[e] (silu(Gate[e] x[t]) * (Up[e] x[t])),   e = ids[t, j]
//
// The first kernel leaves w silu(g) u of every slot, the second reads it against the experts' second matrices.  No sort in front: there are at most 64
// tokens, a lane of a wave each, so the tokens of an expert are a ballot.  In between the numbers are fp32 (Stream, F32).  An expert that a token names twice counts with the sum of
// both weights.

constexpr int kFewTokens = 64, kFewTopk = 16, kFewExperts = 1024;

struct ExpertArgs {
  const void* x;         // [T][x_rs]
  const void* ids;       // [T][topk], int32 or int64, through two strides
  const float* weights;  // [T][topk]
  float* act;            // [T topk][I]
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

// The expert of a slot, -1: none of these.  Both widths by words, without a branch between the loads of several slots.
__device__ __forceinline__ int expert_of(const ExpertArgs& p, int t, int j) {
  const int64_t at = (t * p.ids_s0 + j * p.ids_s1) << p.ids_is64;
  const int32_t* const words = static_cast<const int32_t*>(p.ids);
  const int low = words[at], high = words[at + p.ids_is64];
  return low >= 0 && low < p.E && (p.ids_is64 == 0 || high == 0) ? low : -1;
}

// Lane i of the result: the lane of the i-th bit of the mask.
__device__ __forceinline__ int nth_lane(uint64_t mask, int lane) {
  const uint64_t below = (uint64_t{1} << lane) - 1;
  const bool mine = mask >> lane & 1;
  const int to = mine ? __popcll(mask & below) : __popcll(mask) + __popcll(~mask & below);
  return __builtin_amdgcn_ds_permute(to * 4, lane);
}

// silu(g) u; the fast exponential is off by as many roundings as |g|
__device__ __forceinline__ float gated(float g, float u) { return g / (1.0f + expf(-g)) * u; }

constexpr int kUpWaves = 4;
// Pairs of tiles of Gate and Up that share the rows of x, which are most of what comes into LDS where there are 16 of them (64 tokens, 8 of 32 experts, 4096 x 7168:
// two pairs 226 us e2m1, 251 us e4m3, one 306 and 280 us; eight rows, 16 tokens: 131 and 169 us, one 121 and 146 us; all with four waves to K).
template <int W, int R, int SPLIT>
struct UpShape {
  static constexpr int kPairs = R == 16 ? 2 : 1, kColumns = 16 * kPairs * kUpWaves / SPLIT;  // of a workgroup
  static constexpr int kTiles = 2 * kPairs, kBudget = 2 * kUpWaves * stream_bytes(W, R, kTiles) <= 76 * 1024 ? 76 * 1024 : 152 * 1024;  // two workgroups a CU, or one
  static constexpr int kDepth = stream_depth(W, R, kTiles, kUpWaves, kBudget), kLds = kUpWaves * kDepth * stream_bytes(W, R, kTiles);
};

constexpr int kDownTiles = 2;
// An expert's tokens over those of a pass, rounded up, adds up to no more than the slots, and than the experts and the slots over those of a pass.
__host__ __device__ constexpr int64_t down_entries(int64_t slots, int64_t experts, int64_t a_pass) { return slots < experts + slots / a_pass ? slots : experts + slots / a_pass; }
constexpr int kDownWideTokens = 16;  // as many as eight waves have room for the sums of
template <int W, int TOKENS, int WAVES>
struct DownShape {
  static constexpr int kBudget = (WAVES == 8 ? 138 : 108) * 1024;  // the tables of the tokens have to fit beside it
  static constexpr int kDepth = stream_depth(W, 2 * TOKENS, kDownTiles, WAVES, kBudget), kRing = WAVES * kDepth * stream_bytes(W, 2 * TOKENS, kDownTiles);
};

// A workgroup takes kColumns rows of Gate and the same of Up, SPLIT waves share K; of expert blockIdx.y, or where there are more experts than slots of that slot's expert, if
// it is the first to name it; R of its tokens at a time.
template <int T, int W, int R, int SPLIT>
__global__ void __launch_bounds__(64 * kUpWaves) experts_up_kernel(const ExpertArgs p) {
  typedef UpShape<W, R, SPLIT> Shape;
  constexpr int kPairs = Shape::kPairs, kTiles = Shape::kTiles;
  typedef Stream<T, W, R, kTiles, Shape::kDepth> S;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
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
      const bool names = lane < p.T && j0 + i < p.topk && named[i] == e;
      first = names && first < 0 ? token * p.topk + j0 + i : first;
      weight += names ? w[i] : 0.f;
    }
  }
  const uint64_t mask = __ballot(first >= 0);
  if (mask == 0) return;
  if (by_slot && __shfl(first, __builtin_ctzll(mask)) != y) return;
  const int rows = __popcll(mask), token_of = nth_lane(mask, lane);
  const Matrix up = of_expert(p.up, p.up_q, p.up_s, e);
  const int of = wave % SPLIT, n0 = blockIdx.x * Shape::kColumns + wave / SPLIT * 16 * kPairs;  // past the end: nothing is stored
  v4f* const part = reinterpret_cast<v4f*>(lds);  // [waves][tiles][64]
  for (int b = 0; b < rows; b += R) {
    if (b > 0) __syncthreads();
    S s(lds, wave, lane, p.H, p.x, static_cast<uint32_t>((p.T - 1) * p.x_rs + p.H) * 2, p.up.s);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) s.tile[2 * i].point_at(up, n0 + 16 * i), s.tile[2 * i + 1].point_at(up, p.I + n0 + 16 * i);
#pragma unroll
    for (int j = 0; j < S::kXLoads; ++j) {
      const int i = b + S::x_row(lane, j);
      const int t = __shfl(token_of, i & 63);
      s.set_row(lane, j, i < rows ? static_cast<uint32_t>(t * p.x_rs) * 2 : kNowhere);
    }
    s.split_k(lane, of, SPLIT);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kTiles; ++n) part[(kTiles * wave + n) * 64 + lane] = s.acc[n];
    __syncthreads();
    static_assert(kPairs <= SPLIT, "a wave for each");
    if (of >= kPairs || n0 + 16 * of >= p.I) continue;
    const v4f* const mine = part + (kTiles * (wave - of) + 2 * of) * 64;
    v4f g = mine[lane], u = mine[64 + lane];
#pragma unroll
    for (int w = 1; w < SPLIT; ++w) g += mine[kTiles * w * 64 + lane], u += mine[(kTiles * w + 1) * 64 + lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = b + 4 * q + r;
      const int t = __shfl(token_of, i & 63);
      const int slot = __shfl(first, t);
      const float v = gated(g[r], u[r]) * __shfl(weight, t);
      if (4 * q + r < R && i < rows) p.act[static_cast<int64_t>(slot) * p.I + n0 + 16 * of + l16] = v;
    }
  }
}

// A workgroup takes 32 columns of the output of all tokens.  Its work is a list of experts, several times where one has more than TOKENS of them, by
// chunks of their K = I; each wave takes a run of that and adds its sums up in an LDS table of its own, and the tables are added in wave order.
template <int TO, int W, int TOKENS, int kWaves>
__global__ void __launch_bounds__(64 * kWaves) experts_down_kernel(const ExpertArgs p) {
  constexpr int R = 2 * TOKENS;
  typedef DownShape<W, TOKENS, kWaves> Shape;
  typedef Stream<kInBf16, W, R, kDownTiles, Shape::kDepth, true> S;
  constexpr int kWide = 16 * kDownTiles;
  // The rings; behind them [waves][T][kWide] sums, the entries (expert, pass << 16), the slots of their rows ([TOKENS], -1: none).  What the list of entries is made
  // from lies where the rings are later.
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int entries;
  int* const count = reinterpret_cast<int*>(lds);                                             // [E]
  int16_t(*const ids)[kFewTokens] = reinterpret_cast<int16_t(*)[kFewTokens]>(lds + kFewExperts * 4);  // [topk]
  static_assert(Shape::kRing >= kFewExperts * 4 + kFewTopk * kFewTokens * 2, "room for them");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  const int slots = p.T * p.topk;
  constexpr int kThreads = 64 * kWaves;
  float* const all = reinterpret_cast<float*>(lds + Shape::kRing);
  float* const sums = all + wave * p.T * kWide;
  int32_t* const entry = reinterpret_cast<int32_t*>(all + kWaves * p.T * kWide);
  int16_t* const row_slot = reinterpret_cast<int16_t*>(entry + down_entries(p.T * p.topk, p.E, TOKENS));
  for (int i = tid; i < p.E; i += kThreads) count[i] = 0;
  for (int i = lane; i < p.T * kWide; i += 64) sums[i] = 0.f;
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
      const int passes = e0 + lane < p.E ? (count[e0 + lane] + TOKENS - 1) / TOKENS : 0;
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
  // the rows of every entry, by the waves in turn
  const int count_of_entries = __builtin_amdgcn_readfirstlane(entries);
  for (int i = wave; i < count_of_entries; i += kWaves) {
    const int en = __builtin_amdgcn_readfirstlane(entry[i]), e = en & 0xffff;
    int slot = -1;
    for (int j0 = 0; j0 < p.topk; j0 += 8) {
      int named[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) named[j] = ids[min(j0 + j, p.topk - 1)][lane];
      int at = -1;
#pragma unroll
      for (int j = 7; j >= 0; --j) at = named[j] == e && j0 + j < p.topk ? j0 + j : at;
      if (slot < 0 && at >= 0) slot = lane * p.topk + at;
    }
    if (lane >= p.T) slot = -1;
    const uint64_t mask = __ballot(slot >= 0);
    // row of the lane's token in this pass; rows without one behind the last
    const int row = __popcll(mask & ((uint64_t{1} << lane) - 1)) - (en >> 16) * TOKENS, rows = __popcll(mask) - (en >> 16) * TOKENS;
    if (slot >= 0 && row >= 0 && row < TOKENS) row_slot[i * TOKENS + row] = static_cast<int16_t>(slot);
    if (lane < TOKENS && lane >= rows) row_slot[i * TOKENS + lane] = -1;
  }
  __syncthreads();
  const int n0 = blockIdx.x * kWide;
  S s(lds, wave, lane, p.I, p.act, static_cast<uint32_t>(slots) * p.I * 4, p.down.s);
  const int total = count_of_entries * s.chunks, each = (total + kWaves - 1) / kWaves;
  const int start = min(total, wave * each), end = min(total, start + each);
  auto point_at = [&](int i) {
    const int e = __builtin_amdgcn_readfirstlane(entry[i]) & 0xffff;
#pragma unroll
    for (int j = 0; j < S::kXLoads; ++j) {
      const int slot = row_slot[i * TOKENS + S::x_row(lane, j)];
      s.set_row(lane, j, slot >= 0 ? static_cast<uint32_t>(slot) * p.I * 4 : kNowhere);
    }
#pragma unroll
    for (int n = 0; n < kDownTiles; ++n) s.tile[n].point_at(of_expert(p.down, p.down_q, p.down_s, e), n0 + 16 * n);
  };
  // the chunk that is asked for next, and the one that is multiplied next
  int l_entry = start / s.chunks, l_chunk = start - l_entry * s.chunks, l_left = end - start;
  int m_entry = l_entry, m_chunk = l_chunk, m_left = l_left;
  auto load_next = [&](int d) {
    s.load(d, lane, l_chunk, l_left > 0);
    if (--l_left > 0 && ++l_chunk == s.chunks) l_chunk = 0, point_at(++l_entry);
  };
  // the sums of an entry's rows go to their tokens
  auto leave = [&](int i) {
#pragma unroll
    for (int n = 0; n < kDownTiles; ++n) {
      auto& a = s.sums[n];
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // number r of the first quarter's lanes, from those rows of each turn: row 4 q + r of turn 4 q / TOKENS
        const auto whole = [&](const v4f (&of)[S::kTurns]) {
          if (TOKENS == 2) {
            const float two = of[0][r & 1] + of[1][2 + (r & 1)];
            return S::kTurns == 2 ? two : two + (__shfl_xor(of[S::kTurns - 2][r & 1], 16) + __shfl_xor(of[S::kTurns - 1][2 + (r & 1)], 16));
          }
          if (TOKENS == 8) return of[0][r] + __shfl_xor(of[1][r], 32);
          const float two = of[0][r] + __shfl_xor(of[1][r], 16);
          return S::kTurns == 2 ? two : two + (__shfl_xor(of[S::kTurns - 2][r], 32) + __shfl_xor(of[S::kTurns - 1][r], 48));
        };
        const float first = whole(a.first), rest = whole(a.rest);
        v[r] = fabsf(first) < __builtin_inff() ? first + rest : first;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 4 * q + r, slot = row < TOKENS ? row_slot[i * TOKENS + row] : -1;
        if (slot >= 0) sums[slot / p.topk * kWide + 16 * n + l16] += v[r];
      }
      a.clear();
    }
  };
  if (start < end) {
    point_at(l_entry);
#pragma unroll
    for (int d = 0; d < Shape::kDepth; ++d) {
      load_next(d);
      __builtin_amdgcn_sched_barrier(0);
    }
    for (int i = start; i < end; i += Shape::kDepth) {
#pragma unroll
      for (int d = 0; d < Shape::kDepth; ++d) {
        s.multiply(d, m_chunk);
        if (m_left > 0 && (--m_left == 0 || ++m_chunk == s.chunks)) {
          leave(m_entry);
          m_chunk = 0, ++m_entry;
        }
        load_next(d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    wait_loads<0>();  // nothing is on its way into LDS when the workgroup ends
  }
  __syncthreads();
  for (int i = tid; i < p.T * kWide; i += kThreads) {
    float v = all[i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += all[w * p.T * kWide + i];
    const int t = i / kWide, col = n0 + i % kWide;
    if (col < p.H) store1(p.out, TO, static_cast<int64_t>(t) * p.H + col, v);
  }
}

template <int W, int TOKENS, int WAVES>
int64_t experts_down_lds(int64_t tokens, int64_t topk, int64_t experts) {
  typedef DownShape<W, TOKENS, WAVES> Shape;
  constexpr int kMostTokens = WAVES == 8 ? kDownWideTokens : kFewTokens, kMostSlots = kMostTokens * kFewTopk;
  static_assert(Shape::kRing + WAVES * kMostTokens * 16 * kDownTiles * 4 + kMostSlots * (4 + TOKENS * 2) + 64 <= 160 * 1024, "what a CU has, for the most tokens and slots");
  return Shape::kRing + WAVES * tokens * 16 * kDownTiles * 4 + down_entries(tokens * topk, experts, TOKENS) * (4 + TOKENS * 2);
}

}  // namespace dlb
