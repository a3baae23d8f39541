// Microscaled 4-bit floating point for gfx950: the quantiser and the products of two quantised operands.
//
//   groups of 32 columns of a row share the scale 2^(s - 127), s a byte, 255 = NaN; an element is e2m1, 0 .5 1 1.5 2 3 4 6 with a sign
//   quantising:  s = max(floor(log2 max |x|) - 2, -127) + 127,  q = x 2^(127 - s) to nearest, ties to even, at most 6
//   product:     y[m, n] = sum over the groups g of 2^(a_s[m, g] + b_s[n, g] - 254) sum_{k in g} a[m, k] b[n, k]
//
// (The OCP microscaling formats, version 1.0, name both.)  v_mfma_scale_f32_..._f8f6f4 takes 32 elements and their scale byte from each lane,
// so a group is what one lane holds of one MFMA: 16 bytes of codes, one byte of scales, and which of a chunk's groups goes to which
// lane and step is free as long as both operands agree.  Every kernel here gives a lane neighbouring groups, whose scales are one dword
// and are picked by the instruction's byte selector.  Products of two codes and sums of a group are exact in fp32 (at most 32 x 36 in steps of a
// quarter); the sum over groups is rounded as the unit does it.
#pragma once

#include "rows.h"

namespace dlb {

constexpr int kMxGroup = 32;                // columns
constexpr uint32_t kNowhere = 0x80000000u;  // past the end of every buffer: such a load costs no traffic and gives zero

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}

// ---- quantiser --------------------------------------------------------------------------------------------------------

struct MxQuantArgs {
  const void* x;
  uint32_t* q;   // [rows][K / 2], eight codes a word
  uint8_t* s;    // [rows][K / 32]
  int64_t rows, x_rs;
  int K;
};

// Eight columns a lane, four lanes a group.
template <int T>
__global__ void __launch_bounds__(256) mxfp4_quant_kernel(const MxQuantArgs p) {
  const int64_t per_row = p.K / 8, total = p.rows * per_row;
  const int64_t i = static_cast<int64_t>(blockIdx.y * static_cast<int64_t>(gridDim.x) + blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;  // whole groups
  const int64_t row = i / per_row;
  const int col = static_cast<int>(i - row * per_row) * 8;
  float v[8];
  quant_unpack8<T>(load_raw8<T, true>(p.x, row * p.x_rs, col, 8), v);
  uint32_t top = 0;  // the largest magnitude as bits, which put infinity above all numbers and NaN above infinity
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
  const int exponent = static_cast<int>(top >> 23);  // floor(log2) + 127; 0 of a subnormal number, whose group takes the smallest scale
  const int s = exponent == 255 ? 255 : max(exponent - 2, 0);
  const float up = __uint_as_float(static_cast<uint32_t>(254 - min(s, 253)) << 23);
  uint32_t word = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // the largest is below 8 here; what lies above 6 is 6
    const float a = __builtin_amdgcn_fmed3f(v[2 * k] * up, -6.f, 6.f), b = __builtin_amdgcn_fmed3f(v[2 * k + 1] * up, -6.f, 6.f);
    word |= (__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, a, b, 1.0f, 0) & 0xffu) << (8 * k);
  }
  p.q[i] = s == 255 ? 0 : word;
  if ((threadIdx.x & 3) == 0) p.s[i / 4] = static_cast<uint8_t>(s);
}

// ---- products ---------------------------------------------------------------------------------------------------------

// 16 x 16 outputs, 128 columns: lane l supplies row l % 16 of each operand, 32 consecutive codes, and receives D[4 (l / 16) + r][l % 16] in
// component r.  STEP: byte of the scale words.
template <int STEP>
__device__ __forceinline__ v4f mfma_mx(const v4i& a, uint32_t a_s, const v4i& b, uint32_t b_s, const v4f& c) {
  const v8i aw{a.x, a.y, a.z, a.w, 0, 0, 0, 0}, bw{b.x, b.y, b.z, b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(aw, bw, c, 4, 4, STEP, static_cast<int>(a_s), STEP, static_cast<int>(b_s));
}

// The same for a step that unrolling makes a constant.
__device__ __forceinline__ v4f mfma_mx_step(int step, const v4i& a, uint32_t a_s, const v4i& b, uint32_t b_s, const v4f& c) {
  return step == 0 ? mfma_mx<0>(a, a_s, b, b_s, c) : step == 1 ? mfma_mx<1>(a, a_s, b, b_s, c) : step == 2 ? mfma_mx<2>(a, a_s, b, b_s, c) : mfma_mx<3>(a, a_s, b, b_s, c);
}

struct MxArgs {
  const uint8_t* a;    // [M][K / 2]
  const uint8_t* b;    // [N][K / 2]
  const uint8_t* a_s;  // [M][a_pitch]
  const uint8_t* b_s;  // [N][b_pitch]
  void* c;             // [M][N]
  int64_t M;
  int N, K, G;         // G = K / 32
  int pitch;           // bytes of a row of scales: G, or of scales that were laid out anew
  int out;             // DLB_IN_*
  int tiles_m, tiles_n, group_m;
};

// Four consecutive columns of one row of c.
__device__ __forceinline__ void store4(void* c, int type, int64_t at, const v4f& v, int left) {
  typedef _Float16 v4h_t __attribute__((ext_vector_type(4)));
  if (type == kInF32) {
    float* to = static_cast<float*>(c) + at;
    if (left >= 4) {
      *reinterpret_cast<v4f_el*>(to) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < left) to[i] = v[i];
    }
    return;
  }
  uint16_t* to = static_cast<uint16_t*>(c) + at;
  const v2i h = type == kInBf16 ? __builtin_bit_cast(v2i, __builtin_convertvector(v, v4bf)) : __builtin_bit_cast(v2i, __builtin_convertvector(v, v4h_t));
  typedef v2i v2i_el __attribute__((aligned(2)));
  if (left >= 4) {
    *reinterpret_cast<v2i_el*>(to) = h;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < left) to[i] = static_cast<uint16_t>(static_cast<uint32_t>(h[i / 2]) >> (16 * (i & 1)));
  }
}

// Scales of rows whose groups are no multiple of four, with zeros behind the last: both operands' in one launch.
struct MxPadArgs {
  const uint8_t *a_s, *b_s;
  uint32_t *a_to, *b_to;
  int64_t M, N;
  int G, words;
};
__global__ void __launch_bounds__(256) mxfp4_pad_kernel(const MxPadArgs p) {
  const int64_t total = (p.M + p.N) * p.words;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / p.words;
    const int g = static_cast<int>(i - row * p.words) * 4;
    const uint8_t* from = (row < p.M ? p.a_s + row * p.G : p.b_s + (row - p.M) * p.G) + g;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (g + k < p.G) w |= static_cast<uint32_t>(from[k]) << (8 * k);
    (row < p.M ? p.a_to + row * p.words : p.b_to + (row - p.M) * p.words)[g / 4] = w;
  }
}

// Tiles of BM x BN through LDS.  A step is 128 columns, 64 bytes of every row, in a ring of four; the scales of four steps lie in a table of 16
// bytes a row, two of them in turn.  WGM x WGN waves, each with MF x NF fragments of 16 x 16 outputs (both even).  Bound by what a CU brings into its LDS, about
// 32 KB a microsecond with one or two workgroups on it; a ring of eight takes as long.
template <int WGM_, int WGN_, int MF_, int NF_>
struct MxTile {
  static constexpr int WGM = WGM_, WGN = WGN_, MF = MF_, NF = NF_, STAGES = 4;
  static constexpr int WAVES = WGM * WGN, BM = WGM * MF * 16, BN = WGN * NF * 16;
  static constexpr int A_INST = BM / 16 / WAVES, B_INST = BN / 16 / WAVES;  // an instruction moves 16 rows
  static constexpr int S_INST = (BM + BN) / 64 / WAVES;                      // ... or the scales of 64
  static constexpr int STAGE = (BM + BN) * 64, TABLE = (BM + BN) * 16;
  static constexpr int LDS = STAGES * STAGE + 2 * TABLE;
  static_assert(BM % (16 * WAVES) == 0 && BN % (16 * WAVES) == 0 && (BM + BN) % (64 * WAVES) == 0 && BM % 64 == 0 && LDS <= 160 * 1024, "whole instructions");
};

// Row of a wave's operand that lane or result index i (0 .. 15) of fragment f stands for: two results of a pair of fragments are 8
// consecutive rows, which are 8 consecutive columns of c.
__device__ __forceinline__ int mx_row(int f, int i) { return (f >> 1) * 32 + (f & 1) * 4 + (i >> 2) * 8 + (i & 3); }
// A row's 16-byte chunk c lies at c ^ mx_swizzle(row).  A ds_read_b128 goes through the banks in turns of 16 lanes, lanes 0-3, 12-15 and 20-27 in
// the first, the rest of 0-31 in the second: rows of a fragment's runs g = 0, 3 with one chunk and g = 1, 2 with the next.  Rows are 64
// bytes, so four neighbours fill the banks and what the runs have to differ in is the chunk: (0, 2, 3, 1) does for both turns.
__device__ __forceinline__ int mx_swizzle(int row) {
  const int g = (row >> 3) & 3;
  return (((g ^ (g >> 1)) & 1) << 1) | (g >> 1);
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 0xF) | (((N >> 4) & 0x3) << 14) | (0x7 << 4) | (0xF << 8));
}

// Behind it every wave's LDS reads have returned; loads into LDS stay on their way.
__device__ __forceinline__ void mx_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

typedef __attribute__((address_space(3))) void* mx_lds_ptr;
typedef __attribute__((address_space(3))) uint8_t* mx_lds_bytes;

// Lane i moves 16 bytes to `to` + 16 i.
template <int POLICY, class LdsPtr>
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t src, LdsPtr to, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (mx_lds_ptr)to, 16, voff, soff, 0, POLICY);
}
// ... 4 bytes to `to` + 4 i.
template <class LdsPtr>
__device__ __forceinline__ void load4_to_lds(__amdgpu_buffer_rsrc_t src, LdsPtr to, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (mx_lds_ptr)to, 4, voff, soff, 0, 0);
}

// RAGGED: rows of scales are no whole words.  They go through registers on their way into the table, shifted and with zeros behind the last, instead of being
// laid out anew by a launch of its own.
template <class Tile, bool RAGGED>
__global__ void __launch_bounds__(64 * Tile::WAVES) mxfp4_tile_kernel(const MxArgs p) {
  constexpr int BM = Tile::BM, BN = Tile::BN, MF = Tile::MF, NF = Tile::NF;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const mx_lds_bytes lds = (mx_lds_bytes)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  // neighbouring tiles on one XCD, patches of group_m row tiles
  const int tiles = p.tiles_m * p.tiles_n;
  const int per = tiles / 8, over = tiles % 8, xcd = blockIdx.x % 8;
  const int id = xcd * per + min(xcd, over) + blockIdx.x / 8;
  const int width = p.group_m * p.tiles_n, patch = id / width, first_m = patch * p.group_m;
  const int high = min(p.tiles_m - first_m, p.group_m), in_patch = id - patch * width;
  const int64_t m0 = static_cast<int64_t>(first_m + in_patch % high) * BM;
  const int n0 = (in_patch / high) * BN;
  const int rows = static_cast<int>(min(p.M - m0, static_cast<int64_t>(BM))), cols = min(BN, p.N - n0);
  const uint32_t half = p.K / 2;
  const int steps = (p.G + 3) / 4;

  // 16-byte chunk (lane % 4) of row (lane / 4) of an instruction's 16: where it goes decides what it takes
  const uint8_t *const a_base = p.a + m0 * half, *const b_base = p.b + static_cast<int64_t>(n0) * half;
  uint32_t a_off[Tile::A_INST], b_off[Tile::B_INST], chunk_col;
  {
    const int r = wave * 16 + (lane >> 2);  // of every instruction mod 32: WAVES is even
    chunk_col = static_cast<uint32_t>((lane & 3) ^ mx_swizzle(r)) * 16;
#pragma unroll
    for (int j = 0; j < Tile::A_INST; ++j) a_off[j] = (j * Tile::WAVES * 16 + r) * half + chunk_col;
#pragma unroll
    for (int j = 0; j < Tile::B_INST; ++j) b_off[j] = (j * Tile::WAVES * 16 + r) * half + chunk_col;
  }
  const bool tail = p.G % 4 != 0;  // the last step is short
  auto load_stage = [&](int k) {
    const bool in = k < steps;
    const uint32_t at = in ? static_cast<uint32_t>(k) * 64 : 0;
    const auto a_src = make_rsrc(a_base, in ? rows * half : 0), b_src = make_rsrc(b_base, in ? cols * half : 0);
    const bool past = tail && at + chunk_col >= half;
    const mx_lds_bytes to = lds + (k & 3) * Tile::STAGE;
#pragma unroll
    for (int j = 0; j < Tile::A_INST; ++j)
      load_to_lds<0>(a_src, to + (j * Tile::WAVES + wave) * 1024, past ? kNowhere : a_off[j], at);
#pragma unroll
    for (int j = 0; j < Tile::B_INST; ++j)
      load_to_lds<0>(b_src, to + BM * 64 + (j * Tile::WAVES + wave) * 1024, past ? kNowhere : b_off[j], at);
  };
  // the scales of window w, 16 groups: those of the tile's rows, behind them those of its columns
  uint32_t words[Tile::S_INST][5];
  // RAGGED: of a wave's j-th 64 rows of scales, the word where the operand's start, and from there the lane's row and the end
  struct ScaleRows {
    const uint8_t* base;
    uint32_t at, bytes;
  };
  const auto scale_rows = [&](int j) {
    const int first = (j * Tile::WAVES + wave) * 64;
    const bool of_a = first < BM;
    const uint8_t* const base = of_a ? p.a_s + m0 * p.G : p.b_s + static_cast<int64_t>(n0) * p.G;
    const uint32_t over = reinterpret_cast<uintptr_t>(base) & 3;
    return ScaleRows{base - over, over + (static_cast<uint32_t>(of_a ? first : first - BM) + lane) * p.G, over + static_cast<uint32_t>(of_a ? rows : cols) * p.G};
  };
  auto load_scales = [&](int w) {
    const bool in = 4 * w < steps;
    if (RAGGED) {
#pragma unroll
      for (int j = 0; j < Tile::S_INST; ++j) {
        const ScaleRows r = scale_rows(j);
        const auto src = make_rsrc(r.base, in ? (r.bytes + 3) & ~3u : 0);  // whole words, the last with up to three bytes of something else
        const uint32_t from = (r.at + 16 * w) & ~3u;
        const v4i four = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(src, from, 0, 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) words[j][i] = four[i];
        words[j][4] = __builtin_amdgcn_raw_buffer_load_b32(src, from + 16, 0, 0);
      }
      return;
    }
    const mx_lds_bytes to = lds + Tile::STAGES * Tile::STAGE + (w & 1) * Tile::TABLE;
#pragma unroll
    for (int j = 0; j < Tile::S_INST; ++j) {
      const int first = (j * Tile::WAVES + wave) * 64;
      const bool of_a = first < BM;
      const auto src = make_rsrc(of_a ? p.a_s + m0 * p.pitch : p.b_s + static_cast<int64_t>(n0) * p.pitch, in ? (of_a ? rows : cols) * p.pitch : 0);
      load_to_lds<0>(src, to + first * 16, ((of_a ? first : first - BM) + lane) * static_cast<uint32_t>(p.pitch), in ? 16 * w : 0);
    }
  };

  auto store_scales = [&](int w) {
#pragma unroll
    for (int j = 0; j < Tile::S_INST; ++j) {
      const uint32_t shift = scale_rows(j).at & 3;
      v4i v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int left = p.G - 16 * w - 4 * i;
        v[i] = __builtin_amdgcn_alignbyte(words[j][i + 1], words[j][i], shift) & (left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1);
      }
      *reinterpret_cast<v4i*>(smem + Tile::STAGES * Tile::STAGE + (w & 1) * Tile::TABLE + ((j * Tile::WAVES + wave) * 64 + lane) * 16) = v;
    }
  };

  const int wm = (wave / Tile::WGN) * MF * 16, wn = (wave % Tile::WGN) * NF * 16;
  // a lane's chunk of its row of a fragment; fragments of a pair are 4 rows apart, pairs 32
  const int r0 = mx_row(0, l16);
  const int frag = r0 * 64 + ((q ^ mx_swizzle(r0)) * 16);
  v4f acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  // The scales of a row's 16 groups; a quarter's lane keeps those of its group of each of the four steps, a byte a step.
  const uint32_t pick = 0x04000400u + 0x00010001u * (0x100u * q + q);  // bytes q, 4 + q
  auto own_scales = [&](const uint8_t* row) {
    const v4i v = *reinterpret_cast<const v4i*>(row);
    const uint32_t low = __builtin_amdgcn_perm(v[1], v[0], pick), high = __builtin_amdgcn_perm(v[3], v[2], pick);
    return __builtin_amdgcn_perm(high, low, 0x05040100u);
  };
  uint32_t as[MF], bs[NF];

  load_scales(0);
  if (RAGGED) store_scales(0);
  load_stage(0), load_stage(1), load_stage(2);
  constexpr int kGroup = Tile::A_INST + Tile::B_INST;
  for (int k0 = 0; k0 < steps; k0 += 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + j;
      if (k >= steps) break;
      // in order: what is behind stage k is two stages, and the next scales if they were asked for in between (RAGGED: wherever the compiler put those)
      if (!RAGGED && (j == 1 || j == 2))
        wait_loads<2 * kGroup + Tile::S_INST>();
      else
        wait_loads<2 * kGroup>();
      mx_barrier();
      if (j == 0) load_scales(k / 4 + 1);
      load_stage(k + 3);
      const uint8_t* const stage = smem + (k & 3) * Tile::STAGE;
      const uint8_t* const table = smem + Tile::STAGES * Tile::STAGE + ((k >> 2) & 1) * Tile::TABLE;
      if (j == 0) {
#pragma unroll
        for (int i = 0; i < MF; ++i) as[i] = own_scales(table + (wm + (i >> 1) * 32 + (i & 1) * 4 + r0) * 16);
#pragma unroll
        for (int i = 0; i < NF; ++i) bs[i] = own_scales(table + (BM + wn + (i >> 1) * 32 + (i & 1) * 4 + r0) * 16);
      }
      v4i af[MF], bf[NF];
#pragma unroll
      for (int i = 0; i < NF; ++i) bf[i] = *reinterpret_cast<const v4i*>(stage + (BM + wn + (i >> 1) * 32 + (i & 1) * 4) * 64 + frag);
#pragma unroll
      for (int i = 0; i < MF; ++i) af[i] = *reinterpret_cast<const v4i*>(stage + (wm + (i >> 1) * 32 + (i & 1) * 4) * 64 + frag);
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[i][n] = mfma_mx_step(j, bf[n], bs[n], af[i], as[i], acc[i][n]);
      if (RAGGED && j == 3) store_scales(k / 4 + 1);  // the other table, which was read for the last time a window ago
    }
  }
  wait_loads<0>();  // nothing is on its way into LDS when the workgroup ends
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int row = wm + mx_row(i, l16);
    if (row >= rows) continue;
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      const int col = wn + (n >> 1) * 32 + (n & 1) * 4 + 8 * q;
      if (col < cols) store4(p.c, p.out, (m0 + row) * p.N + n0 + col, acc[i][n], cols - col);
    }
  }
}

// Few rows, or few tiles: 16 MT x 16 NT outputs in a workgroup whose waves split K, a chunk of 256 columns, 128 bytes of every row, each in turn, and add
// their sums through LDS in wave order.  What a wave takes comes through a ring of its own in LDS, so that whole cache lines are asked for and no wave waits for another.
template <int MT_, int NT_, int WAVES_>
struct MxSplit {
  static constexpr int MT = MT_, NT = NT_, WAVES = WAVES_, FRAGS = MT + NT;
  static constexpr int STAGE = FRAGS * 16 * (128 + 12), MOST = 158 * 1024 / (WAVES * STAGE), DEPTH = MOST > 4 ? 4 : MOST;
  static constexpr int SUMS = WAVES * MT * NT * 1024, RING = WAVES * DEPTH * STAGE, LDS = SUMS > RING ? SUMS : RING;
  static_assert(DEPTH >= 1 && LDS <= 160 * 1024, "what a CU has");
};

// A row's 16-byte piece c lies at c ^ this, as in mx_ring_swizzle, for lanes that read pieces 2 (lane / 16) + step of row lane % 16.
__device__ __forceinline__ int mx_split_swizzle(int row) {
  const int i = row >> 1;
  return (i & 4) | (i & 1) << 1 | (((i >> 1) ^ (i >> 2)) & 1);
}

// Two scales, where `left` of a row begin there: past its end are someone else's, of zeros but perhaps no numbers.
typedef uint16_t mx_two_bytes __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t mx_scales_in_row(int left) { return left >= 2 ? 0xffffu : left == 1 ? 0xffu : 0u; }

// The eight scales of a row's chunk start at any byte: they come as the two or three words they lie in.
template <class Split>
__global__ void __launch_bounds__(64 * Split::WAVES) mxfp4_split_kernel(const MxArgs p) {
  constexpr int MT = Split::MT, NT = Split::NT, FRAGS = Split::FRAGS, WAVES = Split::WAVES, DEPTH = Split::DEPTH;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  // eight column tiles, one for each XCD, by the blocks of rows
  const uint32_t beside = 8 * p.tiles_m, group = blockIdx.x / beside, in_group = blockIdx.x - group * beside;
  const int n0 = static_cast<int>(group * 8 + in_group % 8) * 16 * NT;
  const int64_t m0 = static_cast<int64_t>(in_group / 8) * 16 * MT;
  if (n0 >= p.N) return;
  const int cols = min(16 * NT, p.N - n0), rows = static_cast<int>(min(p.M - m0, static_cast<int64_t>(16 * MT)));
  const uint32_t half = p.K / 2, pitch = p.pitch;
  const uint8_t *const a = p.a + m0 * half, *const b = p.b + static_cast<int64_t>(n0) * half;
  const uint8_t *const a_s = p.a_s + m0 * pitch, *const b_s = p.b_s + static_cast<int64_t>(n0) * pitch;
  const int chunks = (p.G + 7) / 8;

  // Fragments of a first, then those of b; an instruction moves eight rows, half of one, and the scales of a whole one are another's.
  const int r8 = lane >> 3;
  const uint32_t piece[2] = {static_cast<uint32_t>((lane & 7) ^ mx_split_swizzle(r8)) * 16, static_cast<uint32_t>((lane & 7) ^ mx_split_swizzle(8 + r8)) * 16};
  uint32_t from[2 * FRAGS];
#pragma unroll
  for (int j = 0; j < 2 * FRAGS; ++j) from[j] = (8 * (j < 2 * MT ? j : j - 2 * MT) + r8) * half + piece[j & 1];
  const mx_lds_bytes ring_to = (mx_lds_bytes)smem + wave * DEPTH * Split::STAGE;
  const bool words = pitch % 4 == 0;
  const uint32_t row_of = words ? lane >> 1 : lane / 3, word = words ? lane & 1 : lane % 3;
  const uint32_t scales_of = row_of < 16 ? (row_of * pitch & ~3u) + 4 * word : kNowhere;
  constexpr int kLoads = FRAGS * 3;
  const auto load = [&](int d, int c) {
    const bool in = c < chunks;
    const uint32_t at = in ? static_cast<uint32_t>(c) * 128 : 0, at_s = in ? static_cast<uint32_t>(c) * 8 : 0;
    const auto a_src = make_rsrc(a, in ? rows * half : 0), b_src = make_rsrc(b, in ? cols * half : 0);
    const auto as_src = make_rsrc(a_s, in ? (rows * pitch + 3) & ~3u : 0), bs_src = make_rsrc(b_s, in ? (cols * pitch + 3) & ~3u : 0);  // whole words
    const mx_lds_bytes to = ring_to + d * Split::STAGE;
    const bool past[2] = {at + piece[0] >= half, at + piece[1] >= half};  // in a short last chunk
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) load_to_lds<0>(a_src, to + j * 1024, past[j & 1] ? kNowhere : from[j], at);
#pragma unroll
    for (int j = 2 * MT; j < 2 * FRAGS; ++j) load_to_lds<2>(b_src, to + j * 1024, past[j & 1] ? kNowhere : from[j], at);
#pragma unroll
    for (int f = 0; f < FRAGS; ++f) {
      const uint32_t first = 16 * (f < MT ? f : f - MT) * pitch;  // a whole word
      if (lane < 48) load4_to_lds(f < MT ? as_src : bs_src, to + FRAGS * 2048 + f * 192, scales_of == kNowhere ? kNowhere : first + scales_of, at_s);
    }
  };

  v4f acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint8_t* const mine = smem + wave * DEPTH * Split::STAGE + l16 * 128;
  const int at[2] = {((2 * q) ^ mx_split_swizzle(l16)) * 16, ((2 * q + 1) ^ mx_split_swizzle(l16)) * 16};
  const int scales_at = FRAGS * 2048 - l16 * 128 + l16 * (words ? 8 : 12) + (l16 * pitch & 3) + 2 * q;
  auto multiply = [&](int d, int c) {
    wait_loads<(DEPTH - 1) * kLoads>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t* const stage = mine + d * Split::STAGE;
    const uint32_t scaled = mx_scales_in_row(p.G - 8 * c - 2 * q);
    v4i v[FRAGS][2];
    uint32_t s[FRAGS];
#pragma unroll
    for (int f = 0; f < FRAGS; ++f) {
      s[f] = *reinterpret_cast<const mx_two_bytes*>(stage + scales_at + f * 192) & scaled;
#pragma unroll
      for (int h = 0; h < 2; ++h) v[f][h] = *reinterpret_cast<const v4i*>(stage + f * 2048 + at[h]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[m][n] = mfma_mx<0>(v[MT + n][0], s[MT + n], v[m][0], s[m], acc[m][n]);
        acc[m][n] = mfma_mx<1>(v[MT + n][1], s[MT + n], v[m][1], s[m], acc[m][n]);
      }
    // what is read of this place has arrived before its next chunk is asked for
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(d, wave + d * WAVES);
  for (int c = wave; c < chunks; c += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      multiply(d, c + d * WAVES);  // zeros past the last chunk
      load(d, c + (DEPTH + d) * WAVES);
    }
  }
  wait_loads<0>();  // nothing is on its way into LDS any more
  __syncthreads();
  v4f* const part = reinterpret_cast<v4f*>(smem);  // [waves][MT][NT][64]
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) part[((wave * MT + m) * NT + n) * 64 + lane] = acc[m][n];
  __syncthreads();
#pragma unroll
  for (int t = wave; t < MT * NT; t += WAVES) {
    v4f sum = part[t * 64 + lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += part[(w * MT * NT + t) * 64 + lane];
    const int row = 16 * (t / NT) + l16, col = 16 * (t % NT) + 4 * q;
    if (row < rows && col < cols) store4(p.c, p.out, (m0 + row) * p.N + n0 + col, sum, cols - col);
  }
}

// Large products: 256 x 256 outputs in eight waves of 128 x 64, steps of 256 columns, 128 bytes of every row, in a ring of two.  Bound by what moves: the MFMAs
// of a step take 2048 cycles (a loop of nothing else reaches 6.3 to 7.3 PFLOP/s on random codes, for its power), its 64 KB come in whole cache lines
// (with steps of half a line, 64-byte requests to the L2, moving them took 280 us of 4096 x 7168 x 18432 without any MFMA).
// LDS is handed over at two points of a step, so that a byte is on its way for one and a half: at Y every wave has read its columns and its first four
// fragments of rows (part one), at X of the next step the other four (part two).  The reads behind a point are covered by the MFMAs of the fragment read
// in front of it.
//   ... X(k): part two of step k + 1 is asked for, fragments 0 to 3 | Y(k): part one of step k + 2, fragments 4 to 7 | X(k + 1) ...
struct MxRing {
  static constexpr int kWaves = 8, kTile = 256, kStage = 2 * kTile * 128, kTable = 2 * kTile * 16, kLds = 2 * kStage + 2 * kTable;
};

// A row's 16-byte piece c lies at c ^ this: as mx_swizzle, of rows of 128 bytes.  Row bit 1 parts neighbours of one parity, and the four runs of a fragment, two of
// which read the next piece in the same turn, take 0, 4, 5, 1.
__device__ __forceinline__ int mx_ring_swizzle(int row) {
  const int g = (row >> 3) & 3;
  return (row & 2) | (((g ^ (g >> 1)) & 1) << 2) | (g >> 1);
}

template <int OUT>
__global__ void __launch_bounds__(64 * MxRing::kWaves) mxfp4_ring_kernel(const MxArgs p) {
  constexpr int kTile = MxRing::kTile;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const mx_lds_bytes lds = (mx_lds_bytes)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4, l16 = lane & 15;
  // neighbouring tiles on one XCD, patches of group_m row tiles
  const int tiles = p.tiles_m * p.tiles_n;
  const int per = tiles / 8, over = tiles % 8, xcd = blockIdx.x % 8;
  const int id = xcd * per + min(xcd, over) + blockIdx.x / 8;
  const int width = p.group_m * p.tiles_n, patch = id / width, first_m = patch * p.group_m;
  const int high = min(p.tiles_m - first_m, p.group_m), in_patch = id - patch * width;
  const int64_t m0 = static_cast<int64_t>(first_m + in_patch % high) * kTile;
  const int n0 = (in_patch / high) * kTile;
  const int rows = static_cast<int>(min(p.M - m0, static_cast<int64_t>(kTile))), cols = min(kTile, p.N - n0);
  const uint32_t half = p.K / 2;
  const int steps = (p.G + 7) / 8;

  // An instruction moves 8 rows, number 8 j + wave of an operand; of the rows, which come in two parts, numbers 0-7 and 16-23, then the others.  All numbers of a
  // wave agree mod 4, which makes the lane's piece the same.
  const uint8_t *const a_base = p.a + m0 * half, *const b_base = p.b + static_cast<int64_t>(n0) * half;
  const uint32_t piece = static_cast<uint32_t>((lane & 7) ^ mx_ring_swizzle(8 * wave + (lane >> 3))) * 16;
  uint32_t a_off[4], b_off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b_off[j] = (64 * j + 8 * wave + (lane >> 3)) * half + piece;
    a_off[j] = (128 * (j & 1) + 64 * (j >> 1) + 8 * wave + (lane >> 3)) * half + piece;
  }
  const bool tail = p.G % 8 != 0;  // the last step is short
  const auto load = [&](bool part_one, int k) {
    const bool in = k < steps;
    const uint32_t at = in ? static_cast<uint32_t>(k) * 128 : 0;
    const bool past = tail && at + piece >= half;
    const auto a_src = make_rsrc(a_base, in ? rows * half : 0), b_src = make_rsrc(b_base, in ? cols * half : 0);
    const mx_lds_bytes to = lds + (k & 1) * MxRing::kStage;
    if (part_one) {
#pragma unroll
      for (int j = 0; j < 4; ++j) load_to_lds<0>(b_src, to + kTile * 128 + (8 * j + wave) * 1024, past ? kNowhere : b_off[j], at);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = part_one ? j : 2 + j;
      load_to_lds<0>(a_src, to + (16 * j + (part_one ? 0 : 8) + wave) * 1024, past ? kNowhere : a_off[i], at);
    }
  };
  // the scales of window w, 16 groups, two steps: those of the tile's rows, behind them those of its columns
  const auto load_scales = [&](int w) {
    const bool in = 2 * w < steps, of_a = wave < 4;
    const auto src = make_rsrc(of_a ? p.a_s + m0 * p.pitch : p.b_s + static_cast<int64_t>(n0) * p.pitch, in ? (of_a ? rows : cols) * p.pitch : 0);
    load_to_lds<0>(src, lds + 2 * MxRing::kStage + (w & 1) * MxRing::kTable + wave * 1024, ((wave & 3) * 64 + lane) * static_cast<uint32_t>(p.pitch), in ? 16 * w : 0);
  };

  const int wm = (wave / 4) * 128, wn = (wave % 4) * 64;
  const int r0 = mx_row(0, l16);
  const int from_a = (wm + r0) * 128 + (q ^ mx_ring_swizzle(r0)) * 16, from_b = (kTile + wn + r0) * 128 + (q ^ mx_ring_swizzle(r0)) * 16;
  struct Fragment {
    v4i half[2];
  };
  const auto fragment = [&](int k, int from, int i) {
    const uint8_t* const at = smem + (k & 1) * MxRing::kStage + ((i >> 1) * 32 + (i & 1) * 4) * 128;
    return Fragment{{*reinterpret_cast<const v4i*>(at + from), *reinterpret_cast<const v4i*>(at + (from ^ 64))}};
  };
  const uint32_t pick = 0x04000400u + 0x00010001u * (0x100u * q + q);  // bytes q, 4 + q
  const auto own_scales = [&](int w, int row) {
    const v4i v = *reinterpret_cast<const v4i*>(smem + 2 * MxRing::kStage + (w & 1) * MxRing::kTable + row * 16);
    const uint32_t low = __builtin_amdgcn_perm(v[1], v[0], pick), high = __builtin_amdgcn_perm(v[3], v[2], pick);
    // groups past the end: what lies there are the next row's, which need not be numbers
    const int bytes = (p.G - 16 * w + 3) / 4;
    return __builtin_amdgcn_perm(high, low, 0x05040100u) & (bytes >= 4 ? ~0u : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1);
  };
  v4f acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[i][n] = v4f{0.f, 0.f, 0.f, 0.f};
  uint32_t as[8], bs[4];
  Fragment b[2][4], a[8];

  const auto products = [&](int parity, int i) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < 4; ++n) acc[i][n] = mfma_mx_step(2 * parity + t, b[parity][n].half[t], bs[n], a[i].half[t], as[i], acc[i][n]);
    __builtin_amdgcn_sched_barrier(0);
  };

  load_scales(0), load(true, 0), load(false, 0), load(true, 1);
  wait_loads<8>();
  mx_barrier();
  load(false, 1);
#pragma unroll
  for (int n = 0; n < 4; ++n) b[0][n] = fragment(0, from_b, n), bs[n] = own_scales(0, kTile + wn + mx_row(n, 0) + r0);
  a[0] = fragment(0, from_a, 0);
#pragma unroll
  for (int i = 0; i < 8; ++i) as[i] = own_scales(0, wm + mx_row(i, 0) + r0);
  for (int k0 = 0; k0 < steps; k0 += 2) {
#pragma unroll
    for (int parity = 0; parity < 2; ++parity) {
      const int k = k0 + parity;
      if (k >= steps) break;
#pragma unroll
      for (int i = 0; i < 3; ++i) a[i + 1] = fragment(k, from_a, i + 1), products(parity, i);
      // Y: part two of this step was asked for at X of the last but one; behind it came one part one, with scales where that step was even, and one part two
      if (parity == 0)
        wait_loads<8>();
      else
        wait_loads<9>();
      mx_barrier();
      if (parity == 0) load_scales(k / 2 + 1);
      load(true, k + 2);
#pragma unroll
      for (int i = 3; i < 7; ++i) a[i + 1] = fragment(k, from_a, i + 1), products(parity, i);
      // X of the next step
      if (parity == 0)
        wait_loads<9>();
      else
        wait_loads<8>();
      mx_barrier();
      load(false, k + 2);
#pragma unroll
      for (int n = 0; n < 4; ++n) b[1 - parity][n] = fragment(k + 1, from_b, n);
      a[0] = fragment(k + 1, from_a, 0);
      products(parity, 7);
      if (parity == 1) {
#pragma unroll
        for (int n = 0; n < 4; ++n) bs[n] = own_scales(k / 2 + 1, kTile + wn + mx_row(n, 0) + r0);
#pragma unroll
        for (int i = 0; i < 8; ++i) as[i] = own_scales(k / 2 + 1, wm + mx_row(i, 0) + r0);
      }
    }
  }
  wait_loads<0>();  // nothing is on its way into LDS when the workgroup ends
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = wm + mx_row(i, l16);
    if (row >= rows) continue;
#pragma unroll
    for (int n = 0; n < 4; n += 2) {
      const int col = wn + (n >> 1) * 32 + 8 * q;
      if (col >= cols) continue;
      const float v[8] = {acc[i][n][0], acc[i][n][1], acc[i][n][2], acc[i][n][3], acc[i][n + 1][0], acc[i][n + 1][1], acc[i][n + 1][2], acc[i][n + 1][3]};
      store_raw8<OUT>(p.c, (m0 + row) * p.N + n0, col, pack_raw8<OUT>(v), cols - col);
    }
  }
}

}  // namespace dlb
