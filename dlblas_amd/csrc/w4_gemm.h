// Products of a few rows with 4-bit weights and group scales for gfx950, and the quantiser that makes such weights.
//
//   y[m, n] = sum over the groups g of s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g])        z = 8 without zero points
//
// Both kernels take both layouts: all rows against one matrix, or the rows [row_start[e], row_end[e]) against the matrix of expert e.
// Bound by the weights' bytes while the rows are few, so every weight byte goes from memory to a register once and straight into
// v_mfma_f32_16x16x32: a lane's 16 bytes are 32 weights of one row of the matrix, four MFMA steps.  There is no conversion: a code
// moved to the top of the significand of the float 16 is 16 + q exactly (bf16: bits 3 to 6, fp16: bits 6 to 9), a shift and an
// and-or for two weights, and the 16 leaves through the sum of x over the group:
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x
// in fp32; the scale multiplies that once per group.  The kernel whose waves split K has sum x from an MFMA with a matrix of ones and takes
// (16 + z) times it off; the one whose tiles share x adds -(16 + z) x through an MFMA of its own, which is half of the products it issues.  What this costs is rounding of the fp32 sums of terms up to 31 |x| instead of
// |q - z| |x|: the unit adds the 8 products of a quarter cut off 2^-24 below the largest of them and rounds after each quarter
// (measured with ladders of powers of two), so a group's sum is off by at most 24 * 2^-24 * 62 sum |x|.
// A word's eight codes come out as the pairs (0, 4), (1, 5), (2, 6), (3, 7); x is put into the same order.
// The waves of a workgroup take blocks of 128 columns in turn and add their sums through LDS in wave order at the end.
#pragma once

#include <type_traits>

#include "fp8_gemm_common.h"
#include "fp8_quant.h"
#include "rms_norm.h"

namespace dlb {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct W4Args {
  const void* x;
  const uint8_t* q;          // [E][N][K / 2], low nibble = even column
  const void* s;             // [E][N][G], bf16 or fp16 (s_type)
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

// Zero points are 0 to 15, and 16, which a checkpoint that keeps z - 1 comes to: 16 + z is 32 then, still exact in every form here.  A byte
// above that is none, and its group's scale is taken as NaN, so that its column shows it whichever kernel runs.
constexpr uint32_t kMaxZero = 16;

template <int T>
__device__ __forceinline__ v4f mfma_16x16x32(const v4i& a, const v4i& b, const v4f& c) {
  if (T == kInBf16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const uint8_t* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, bytes, 0x00020000);
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

// The values of a lane's quarter in all quarters: v[i] of the result is what quarter i held.
template <int N>
__device__ __forceinline__ void spread_quarters(float v, float (&out)[N]) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  const unsigned u = __float_as_uint(v);
  if (N == 1) {
    out[0] = v;
    return;
  }
  const v2u h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  if (N == 2) {
    out[0] = __uint_as_float(h[0]), out[N - 1] = __uint_as_float(h[1]);
    return;
  }
  const v2u lo = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false);
  const v2u hi = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
  out[0] = __uint_as_float(lo[0]), out[1 % N] = __uint_as_float(lo[1]), out[2 % N] = __uint_as_float(hi[0]), out[3 % N] = __uint_as_float(hi[1]);
}

// The which-th expert that has rows among those there are, -1: there are not so many.
__device__ __forceinline__ int nth_expert(const W4Args& p, int which, int lane) {
  for (int e0 = 0; e0 < p.E; e0 += 64) {
    const int i = min(e0 + lane, p.E - 1);
    uint64_t some = __ballot(e0 + lane < p.E && min(static_cast<int64_t>(p.row_end[i]), p.rows) > max(p.row_start[i], 0));
    const int n = __popcll(some);
    if (which >= n) {
      which -= n;
      continue;
    }
    for (; which > 0; --which) some &= some - 1;
    return __builtin_amdgcn_readfirstlane(e0 + __builtin_ctzll(some));
  }
  return -1;
}

// Chunks of 256 columns with groups of 128: a quarter holds 64 columns, words of a and then of b.  Afterwards a holds the columns of the
// first group and b those of the second: quarters 0 and 1 keep their place in a, 2 and 3 in b.
__device__ __forceinline__ void exchange_halves(v4i& a, v4i& b) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const v2u h = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);
    a[i] = static_cast<int>(h[0]), b[i] = static_cast<int>(h[1]);
  }
}
// N consecutive values of 1 or 2 bytes in one load at any alignment of theirs.
template <typename E, int N>
__device__ __forceinline__ uint64_t load_packed(const E* p) {
  constexpr int kBytes = sizeof(E) * N;
  typedef std::conditional_t<kBytes == 8, uint64_t, std::conditional_t<kBytes == 4, uint32_t, std::conditional_t<kBytes == 2, uint16_t, uint8_t>>> word;
  typedef word word_el __attribute__((aligned(sizeof(E))));
  return *reinterpret_cast<const word_el*>(p);
}
// Two 16-bit scales of which those are NaN whose zero point, byte 2 J or 2 J + 1 of z, is none: bit 7 of a byte shows it, moved up to bit
// 15 of a half, from where a borrow fills the bits below.
template <int J>
__device__ __forceinline__ uint32_t mark_bad_zeros(uint32_t scales, uint32_t z) {
  const uint32_t over = ((z & 0x7f7f7f7fu) + 0x01010101u * (0x7fu - kMaxZero)) | z;
  const uint32_t top = __builtin_amdgcn_perm(over & 0x80808080u, 0, J == 0 ? 0x050c040cu : 0x070c060cu);
  return scales | (top - (top >> 15));
}
// A word of every lane as the lanes of each half have it, in all lanes of both.
struct Halves {
  uint32_t low, high;
};
__device__ __forceinline__ Halves halves(uint32_t v) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  const v2u h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return {h[0], h[1]};
}
// And as the lanes of each quarter have it; `same`: both quarters of a half hold the same.
__device__ __forceinline__ void quarters(const Halves& h, uint32_t (&out)[4], bool low, bool same, bool high) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  if (same) {
    out[0] = out[1] = h.low, out[2] = out[3] = h.high;
    return;
  }
  if (low) {
    const v2u l = __builtin_amdgcn_permlane16_swap(h.low, h.low, false, false);
    out[0] = l[0], out[1] = l[1];
  }
  if (high) {
    const v2u g = __builtin_amdgcn_permlane16_swap(h.high, h.high, false, false);
    out[2] = g[0], out[3] = g[1];
  }
}

constexpr int kW4Waves = 4;  // of a workgroup, in both kernels

// What a wave reads for one block of 128 columns: its weights, the scale (and zero point) of the quarter's group, its rows of x.
struct W4Block {
  v4i w;
  uint32_t s, z;
  v4i x[4];
};

// GROUPS = groups in a block of 128 columns: 1, 2, 4 for groups of 128, 64, 32.  A tile is 16 rows of x by 16 rows of the
// matrix.  After the exchange of words between the quarters, step i of a block is columns 32 i to 32 i + 31, 8 a quarter.
// kW4Depth blocks are on their way to a wave at a time.  Loads return in the order they were issued in, so all that a block needs is
// asked for together, and none of them stands behind a branch, because a wait counts the loads issued since: what lies outside
// (rows past the tile, columns past the end, blocks past the last one) has an offset past the end of the buffer, which costs no
// traffic and gives zero.  For products whose launch and latency count: 1 x 2112 x 7168 7.0 us (7.8 MB), 5 tokens x 2 of 8 experts x 1000 x 1056
// fp16, groups of 32 with zero points 6.8 us, 1 x 512 x 2048 4.3; two waves instead of four 9.4, 7.6, 4.5, eight 8.6, 12.4, 6.1.
constexpr int kW4Depth = 4;

template <int T, int GROUPS, bool ZEROS>
__global__ void __launch_bounds__(64 * kW4Waves) w4_gemm_kernel(const W4Args p) {
  __shared__ float part[kW4Waves][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int quarter = lane >> 4, l16 = lane & 15;
  constexpr uint32_t kNowhere = 0x80000000u;  // every buffer is shorter
  int64_t expert = 0;
  int64_t row0 = static_cast<int64_t>(blockIdx.y) * 16, row_end = min(p.rows, row0 + 16);
  if (p.row_start) {
    const int e = nth_expert(p, blockIdx.y, lane);
    if (e < 0) return;
    row0 = max(p.row_start[e], 0), row_end = min(static_cast<int64_t>(p.row_end[e]), p.rows);
    expert = e;
  }
  const int blocks = (p.K + 127) / 128;
  const uint32_t half = p.K / 2;  // bytes of a row
  const int n0 = static_cast<int>(blockIdx.x) * 16;
  const int cols = min(16, p.N - n0);
  const uint8_t* w_ptr = p.q + expert * p.q_es + static_cast<int64_t>(n0) * half;
  const int64_t s0 = expert * p.s_es + static_cast<int64_t>(n0) * p.G;
  const uint8_t *s_ptr = static_cast<const uint8_t*>(p.s) + 2 * s0, *z_ptr = ZEROS ? p.z + s0 : p.q;
  const uint32_t w_bytes = cols * half, s_count = cols * p.G;
  const uint32_t w_off = l16 * half + 16 * quarter, s_off = l16 * p.G + quarter * GROUPS / 4;  // of rows past the matrix: past the end
  // in registers, where one v_and_or_b32 takes both
  int mask = T == kInBf16 ? 0x00780078 : 0x03c003c0, bits = T == kInBf16 ? 0x41804180 : 0x4c004c00;
  asm("" : "+s"(mask));
  asm("" : "+v"(bits));
  v4i ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) ones[i] = T == kInBf16 ? 0x3f803f80 : 0x3c003c00;

  for (; row0 < row_end; row0 += 16) {
    const int rows = static_cast<int>(min(row_end - row0, int64_t{16}));
    const uint32_t x_row = static_cast<uint32_t>(p.x_rs) * 2;
    const uint8_t* x_ptr = static_cast<const uint8_t*>(p.x) + row0 * p.x_rs * 2;
    const uint32_t x_bytes = (rows - 1) * x_row + 2u * p.K;
    const uint32_t x_off = l16 < rows ? l16 * x_row + 16 * quarter : kNowhere;
    v4f acc{0.f, 0.f, 0.f, 0.f};
    // The place of a block travels in the scalar offset, so a load costs no vector instruction; past the last block the buffers are
    // empty.  A lane past the last column of a row
    // reads the next row's codes, which then meet zeros of x; the scale of such a group is replaced in multiply().
    auto load = [&](int kb, W4Block& b) {
      const bool in = kb < blocks;
      const uint32_t at = in ? kb : 0;
      const auto w_src = make_rsrc(w_ptr, in ? w_bytes : 0), s_src = make_rsrc(s_ptr, in ? 2 * s_count : 0), z_src = make_rsrc(z_ptr, ZEROS && in ? s_count : 0);
      const auto x_src = make_rsrc(x_ptr, in ? x_bytes : 0);
      b.w = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(w_src, w_off, 64 * at, 2));
      b.s = __builtin_amdgcn_raw_buffer_load_b16(s_src, 2 * s_off, 2 * GROUPS * at, 0);
      if (ZEROS) b.z = __builtin_amdgcn_raw_buffer_load_b8(z_src, s_off, GROUPS * at, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) b.x[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(x_src, x_off + 64 * i, 256 * at, 0));
    };
    auto multiply = [&](int kb, W4Block& b) {
      float sc[GROUPS], coef[GROUPS];
      transpose_quarters(b.w);
      float s = p.s_type == kInBf16 ? __uint_as_float(b.s << 16) : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(b.s)));
      if (ZEROS && b.z > kMaxZero) s = __builtin_nanf("");
      if (GROUPS > 1 && kb * GROUPS + quarter * GROUPS / 4 >= p.G) s = 0.f;
      spread_quarters(s, sc);
      if (ZEROS)
        spread_quarters(-16.f - static_cast<float>(b.z), coef);
      else
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) coef[g] = -24.f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        v4f sum{0.f, 0.f, 0.f, 0.f}, xs{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = g * 4 / GROUPS; i < (g + 1) * 4 / GROUPS; ++i) {
          // columns past the end: what was read there is the next row, and selecting byte 12 gives zero
          const bool in = kb * 128 + 32 * i < p.K;
          const uint32_t low = in ? 0x05040100u : 0x0c0c0c0cu, high = in ? 0x07060302u : 0x0c0c0c0cu;
          const v4i v = b.x[i];
          const v4i xf{static_cast<int>(__builtin_amdgcn_perm(v[2], v[0], low)), static_cast<int>(__builtin_amdgcn_perm(v[2], v[0], high)),
                       static_cast<int>(__builtin_amdgcn_perm(v[3], v[1], low)), static_cast<int>(__builtin_amdgcn_perm(v[3], v[1], high))};
          xs = mfma_16x16x32<T>(xf, ones, xs);
          constexpr int kUp = T == kInBf16 ? 3 : 6;
          const int word = b.w[i];
          v4i codes;
#pragma unroll
          for (int j = 0; j < 4; ++j) codes[j] = ((4 * j < kUp ? word << (kUp - 4 * j) : word >> (4 * j - kUp)) & mask) | bits;
          sum = mfma_16x16x32<T>(xf, codes, sum);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = fmaf(sc[g], fmaf(coef[g], xs[r], sum[r]), acc[r]);
      }
    };
    W4Block on_way[kW4Depth];
#pragma unroll
    for (int d = 0; d < kW4Depth; ++d) {
      load(wave + d * kW4Waves, on_way[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
    for (int kb = wave; kb < blocks; kb += kW4Depth * kW4Waves) {
      // whole turns: blocks past the last one multiply zeros; the order of loads and products stays as it is written
#pragma unroll
      for (int d = 0; d < kW4Depth; ++d) {
        multiply(kb + d * kW4Waves, on_way[d]);
        __builtin_amdgcn_sched_barrier(0);
        load(kb + (kW4Depth + d) * kW4Waves, on_way[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // lane l holds rows 4 (l / 16) + r, column l % 16 of the tile
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][(4 * quarter + r) * 16 + l16] = acc[r];
    __syncthreads();
    const int row = tid / 16, col = tid % 16;  // a thread an element
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kW4Waves; ++w) sum += part[w][tid];
    if (row < rows && col < cols) {
      const int64_t at = (row0 + row) * p.y_rs + n0 + col;
      if (T == kInBf16)
        static_cast<__bf16*>(p.y)[at] = static_cast<__bf16>(sum);
      else
        static_cast<_Float16*>(p.y)[at] = static_cast<_Float16>(sum);
    }
    __syncthreads();
  }
}

// The same product for more than a little work.  Four waves take neighbouring tiles and ask memory for nothing but weights and scales, a
// chunk of UNITS x 256 columns ahead; x goes through LDS once for all of them, in the order in which they read it.
// A lane reads 32 bytes of a unit's 128 bytes of a row in two loads, so a load touches whole cache lines: 64 columns a quarter.
// Eight steps of 32 columns follow, of one group each: for groups of 128 the halves of the wave exchange words, for smaller ones the
// quarters.  Slices of K (gridDim.z) go to workgroups of their own, whose fp32 sums w4_sum_kernel adds in slice order.
// 32 experts x 4 rows x 4096 x 7168, 482 MB: 100 us call after call on three sets of weights, of which the cache keeps some, 119 on weights
// from memory, 4.1 TB/s where streams of weights with the non-temporal bit, which these loads do not have, reach 6.9; 16 x 7168 x 18432, 69 MB
// in nine slices: 20 us and 4 for the sums from memory, instructions of the few waves per SIMD and the start of the stream; 64 x 7168 x 18432 47 us, where a SIMD has 13 us of products and 15
// of other vector instructions to issue and its one or two waves overlap them badly (a third of their time each waiting for issue, waiting for
// LDS and memory, issuing).  Two chunks on their way instead of one 28 and 49 us, three 30 and 52.
constexpr int kW4Unit = 256;  // columns

// PIECES = 16-byte pieces of x a thread moves per chunk: all rows of a tile take 2 MT UNITS, one is enough for 8 / UNITS rows (1 x 7168 x
// 18432 22.9 -> 21.1 us).
template <int T, int GROUPS, bool ZEROS, int MT, int NT, int UNITS, int PIECES>
__global__ void __launch_bounds__(64 * kW4Waves) w4_gemm_shared_kernel(const W4Args p, float* sums, int chunks_each) {
  constexpr int kThreads = 64 * kW4Waves;
  constexpr int kUnitGroups = 2 * GROUPS;
  constexpr int kChunkGroups = kUnitGroups * UNITS;
  constexpr int kMine = kChunkGroups / 4 > 0 ? kChunkGroups / 4 : 1;  // of them a quarter reads the scales of, in one load
  constexpr int kWords = (kMine + 1) / 2;                             // of them
  constexpr int kPitch = 128 * UNITS + 16;     // bytes of a row's steps in LDS, neighbouring rows on other banks
  constexpr int kPlane = 16 * MT * kPitch;     // x of a quarter
  __shared__ __attribute__((aligned(16))) char x_lds[2][4 * kPlane];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int quarter = lane >> 4, l16 = lane & 15;
  constexpr uint32_t kNowhere = 0x80000000u;  // past the end of every buffer
  int64_t expert = 0;
  int64_t row0 = static_cast<int64_t>(blockIdx.y) * 16 * MT, row_end = min(p.rows, row0 + 16 * MT);
  if (p.row_start) {
    const int e = nth_expert(p, blockIdx.y, lane);
    if (e < 0) return;
    row0 = max(p.row_start[e], 0), row_end = min(static_cast<int64_t>(p.row_end[e]), p.rows);
    expert = e;
  }
  constexpr int kColumns = kW4Unit * UNITS;
  const int first = blockIdx.z * chunks_each, last = min((p.K + kColumns - 1) / kColumns, first + chunks_each);
  const uint32_t half = p.K / 2;
  const int n0 = (static_cast<int>(blockIdx.x) * kW4Waves + wave) * 16 * NT;
  const int cols = max(0, min(16 * NT, p.N - n0));
  const int64_t n_base = min(n0, p.N - 1);
  const uint8_t* w_ptr = p.q + expert * p.q_es + n_base * half;
  const int64_t s0 = expert * p.s_es + n_base * p.G;
  const uint16_t* s_ptr = static_cast<const uint16_t*>(p.s) + s0;
  const uint8_t* z_ptr = ZEROS ? p.z + s0 : nullptr;
  const int s_last = static_cast<int>(min(p.E * p.s_es - s0, int64_t{1} << 30)) - kMine;  // where the last load of them can start
  const uint32_t w_bytes = cols * half;
  const int my_group = kChunkGroups < 4 ? quarter >> 1 : quarter * kMine;
  uint32_t w_off[NT];  // of rows past the matrix: past the end
  int s_off[NT];       // of rows past the matrix: the last row's
#pragma unroll
  for (int n = 0; n < NT; ++n) w_off[n] = (16 * n + l16) * half + 32 * quarter, s_off[n] = max(0, min(16 * n + l16, cols - 1)) * p.G + my_group;
  // in registers, where one v_and_or_b32 takes both
  int mask = T == kInBf16 ? 0x00780078 : 0x03c003c0, bits = T == kInBf16 ? 0x41804180 : 0x4c004c00;
  asm("" : "+s"(mask));
  asm("" : "+v"(bits));
  uint32_t s_bf16 = p.s_type == kInBf16 ? ~0u : 0u;
  asm("" : "+v"(s_bf16));
  const char* const x_mine = &x_lds[0][quarter * kPlane + l16 * kPitch];

  struct Chunk {
    v4i w[NT][UNITS][2];
    uint64_t s[NT];  // kMine scales
    uint32_t z[NT];
  };
  auto load = [&](int c, Chunk& b) {
    const bool in = c < last && w_bytes > 0;  // a scalar offset stays below the length of its buffer
    const uint32_t at = in ? c * UNITS : 0;
    const auto w_src = make_rsrc(w_ptr, in ? w_bytes : 0);
    const auto s_src = make_rsrc(reinterpret_cast<const uint8_t*>(s_ptr), in ? 2u * cols * p.G : 0), z_src = make_rsrc(ZEROS ? z_ptr : p.q, ZEROS && in ? cols * p.G : 0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k) b.w[n][u][k] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(w_src, w_off[n] + 128 * u + 16 * k, 128 * at, 0));
      // A load touches 16 cache lines however little it takes of each, and beside the matrices' bytes that is what these kernels wait for:
      // one load for all that the lane needs (32 experts x 4 rows x 4096 x 7168, groups of 32 with zero points, a load for each scale
      // 175 us, so 137).  Near the end of the tensor it starts earlier and the rest moves down in multiply().
      if (kMine == 1) {
        b.s[n] = __builtin_amdgcn_raw_buffer_load_b16(s_src, 2 * s_off[n], 2 * kUnitGroups * at, 0);
        if (ZEROS) b.z[n] = __builtin_amdgcn_raw_buffer_load_b8(z_src, s_off[n], kUnitGroups * at, 0);
      } else {
        const int from = min(s_off[n] + c * kChunkGroups, s_last);
        b.s[n] = load_packed<uint16_t, kMine>(s_ptr + from);
        if (ZEROS) b.z[n] = static_cast<uint32_t>(load_packed<uint8_t, kMine>(z_ptr + from));
      }
    }
  };
  for (; row0 < row_end; row0 += 16 * MT) {
    const int rows = static_cast<int>(min(row_end - row0, static_cast<int64_t>(16 * MT)));
    const uint32_t x_pitch = static_cast<uint32_t>(p.x_rs) * 2;
    const uint8_t* x_ptr = static_cast<const uint8_t*>(p.x) + row0 * p.x_rs * 2;
    const uint32_t x_bytes = (rows - 1) * x_pitch + 2u * p.K;
    // piece j of a thread: 8 columns of row x_r + j rows_apart, for the step and quarter that read them
    constexpr int kRowPieces = 32 * UNITS, kRowsApart = kThreads / kRowPieces;
    const int x_r = tid / kRowPieces, x_col8 = tid % kRowPieces, in_unit = x_col8 & 31;
    const int x_step = GROUPS > 1 ? in_unit >> 2 : 4 * (in_unit >> 4) + (in_unit & 3);
    const int x_quarter = GROUPS > 1 ? in_unit & 3 : ((in_unit >> 3) & 1) + ((in_unit >> 2) & 1) * 2;
    const int x_to = x_quarter * kPlane + x_r * kPitch + (x_col8 >> 5) * 128 + x_step * 16;
    v4i piece[PIECES];
    auto load_x = [&](int c) {
      const auto x_src = make_rsrc(x_ptr, c < last ? x_bytes : 0);
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const int r = x_r + j * kRowsApart;
        piece[j] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(x_src, r < rows ? r * x_pitch + 16 * x_col8 : kNowhere, c < last ? c * (2u * kColumns) : 0, 0));
      }
    };
    auto keep_x = [&](int c, int buf) {
      // columns past the end: what was read there is the next row, and selecting byte 12 gives zero
      const bool in = c * kColumns + 8 * x_col8 < p.K;
      const uint32_t low = in ? 0x05040100u : 0x0c0c0c0cu, high = in ? 0x07060302u : 0x0c0c0c0cu;
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const v4i v = piece[j];
        const v4i o{static_cast<int>(__builtin_amdgcn_perm(v[2], v[0], low)), static_cast<int>(__builtin_amdgcn_perm(v[2], v[0], high)),
                    static_cast<int>(__builtin_amdgcn_perm(v[3], v[1], low)), static_cast<int>(__builtin_amdgcn_perm(v[3], v[1], high))};
        *reinterpret_cast<v4i*>(&x_lds[buf][x_to + j * kRowsApart * kPitch]) = o;
      }
    };
    v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int c, Chunk& b, int buf) {
      // a scale in the upper 16 bits; not by a branch, which would part the products
      const auto widened = [&](uint32_t up) {
        const uint32_t from_half = __float_as_uint(static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(up >> 16))));
        return __uint_as_float((up & s_bf16) | (from_half & ~s_bf16));
      };
      // scales (widened where a lane read one) and zero points, of the quarters 0, 1 and 2, 3 in words of their own
      Halves sh[NT][kWords], zh[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int mine = p.G - (c * kChunkGroups + my_group);  // groups left in the row
        if (kMine == 1) {
          const uint32_t s = ZEROS && b.z[n] > kMaxZero ? 0x7fc00000u : __float_as_uint(widened(static_cast<uint32_t>(b.s[n]) << 16));
          sh[n][0] = halves(mine > 0 ? s : 0u);
          if (ZEROS) zh[n] = halves(b.z[n]);
          continue;
        }
        const int down = max(0, min(s_off[n] + c * kChunkGroups - s_last, kMine - 1));
        uint64_t s = b.s[n] >> (16 * down);
        if (ZEROS) {
          const uint32_t z = b.z[n] >> (8 * down);
          zh[n] = halves(z);
          const uint64_t high = kWords > 1 ? mark_bad_zeros<1>(static_cast<uint32_t>(s >> 32), z) : 0u;
          s = high << 32 | mark_bad_zeros<0>(static_cast<uint32_t>(s), z);
        }
        if (mine < kMine) s &= (uint64_t{1} << (16 * max(0, mine))) - 1;
#pragma unroll
        for (int j = 0; j < kWords; ++j) sh[n][j] = halves(static_cast<uint32_t>(s >> (32 * j)));
      }
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        uint32_t sw[NT][kWords][4], zw[NT][4];  // by quarter; of the unit's alone
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < kWords; ++j) quarters(sh[n][j], sw[n][j], UNITS == 1 || u == 0, kChunkGroups < 4, UNITS == 1 || u == 1);
          if (ZEROS) quarters(zh[n], zw[n], UNITS == 1 || u == 0, kChunkGroups < 4, UNITS == 1 || u == 1);
        }
        const auto scale = [&](int n, int g) {  // g of the chunk
          const int q = kChunkGroups < 4 ? 2 * g : g / kMine, j = kChunkGroups < 4 ? 0 : g % kMine;
          const uint32_t word = sw[n][j / 2][q];
          return kMine == 1 ? __uint_as_float(word) : widened(j % 2 ? word & 0xffff0000u : word << 16);
        };
        // -(16 + z) of a group twice: the matrix through which the constant leaves
        const auto minus = [&](int n, int g) {
          const int q = kChunkGroups < 4 ? 2 * g : g / kMine, j = kChunkGroups < 4 ? 0 : g % kMine;
          const uint32_t z = (zw[n][q] >> (8 * j)) & 0xffu;
          return static_cast<int>(z * (T == kInBf16 ? 0x80008u : 0x400040u) + (static_cast<uint32_t>(bits) | 0x80008000u));
        };
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (GROUPS == 1)
            exchange_halves(b.w[n][u][0], b.w[n][u][1]);
          else
            transpose_quarters(b.w[n][u][0]), transpose_quarters(b.w[n][u][1]);
        }
#pragma unroll
        for (int g = 0; g < kUnitGroups; ++g) {
          v4f sum[MT][NT];
          float sc[NT];
          int constant[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) sc[n] = scale(n, u * kUnitGroups + g), constant[n] = ZEROS ? minus(n, u * kUnitGroups + g) : static_cast<int>(T == kInBf16 ? 0xc1c0c1c0 : 0xce00ce00);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) sum[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = g * 4 / GROUPS; st < (g + 1) * 4 / GROUPS; ++st) {
            v4i xf[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) xf[m] = *reinterpret_cast<const v4i*>(x_mine + buf * 4 * kPlane + m * 16 * kPitch + u * 128 + st * 16);
            constexpr int kUp = T == kInBf16 ? 3 : 6;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int word = GROUPS == 1 ? b.w[n][u][st >> 2][st & 3] : b.w[n][u][st & 1][st >> 1];
              v4i v, c16;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                v[j] = ((4 * j < kUp ? word << (kUp - 4 * j) : word >> (4 * j - kUp)) & mask) | bits;
                c16[j] = constant[n];
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                sum[m][n] = mfma_16x16x32<T>(xf[m], c16, sum[m][n]);
                sum[m][n] = mfma_16x16x32<T>(xf[m], v, sum[m][n]);
              }
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[m][n][r] = fmaf(sc[n], sum[m][n][r], acc[m][n][r]);
        }
      }
    };
    Chunk even, odd;
    load_x(first);
    load(first, even);
    __builtin_amdgcn_sched_barrier(0);
    keep_x(first, 0);
    lds_barrier();
    for (int c = first; c < last; c += 2) {
      // x before the weights: loads return in order.  Past the last chunk: zeros
      load_x(c + 1);
      load(c + 1, odd);
      __builtin_amdgcn_sched_barrier(0);
      multiply(c, even, 0);
      __builtin_amdgcn_sched_barrier(0);
      keep_x(c + 1, 1);
      lds_barrier();
      load_x(c + 2);
      load(c + 2, even);
      __builtin_amdgcn_sched_barrier(0);
      multiply(c + 1, odd, 1);
      __builtin_amdgcn_sched_barrier(0);
      keep_x(c + 2, 0);
      lds_barrier();
    }
    // lane l holds rows 4 (l / 16) + r, column l % 16 of a tile
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * m + 4 * quarter + r, col = 16 * n + l16;
          if (row >= rows || col >= cols) continue;
          if (sums) {
            sums[(blockIdx.z * p.rows + row0 + row) * p.N + n0 + col] = acc[m][n][r];
            continue;
          }
          const int64_t at = (row0 + row) * p.y_rs + n0 + col;
          if (T == kInBf16)
            static_cast<__bf16*>(p.y)[at] = static_cast<__bf16>(acc[m][n][r]);
          else
            static_cast<_Float16*>(p.y)[at] = static_cast<_Float16>(acc[m][n][r]);
        }
  }
}

// y = the sums of the slices of K, added in their order: 4 us of launch and latency for nine slices of 16 x 7168.
template <int T>
__global__ void __launch_bounds__(256) w4_sum_kernel(const float* sums, void* y, int64_t y_rs, int64_t rows, int N, int slices) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * N) return;
  float s = 0.f;
  int z = 0;
  for (; z + 4 <= slices; z += 4) {
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = sums[(z + u) * rows * N + i];
#pragma unroll
    for (int u = 0; u < 4; ++u) s += v[u];
  }
  for (; z < slices; ++z) s += sums[z * rows * N + i];
  const int64_t row = i / N, at = row * y_rs + (i - row * N);
  if (T == kInBf16)
    static_cast<__bf16*>(y)[at] = static_cast<__bf16>(s);
  else
    static_cast<_Float16*>(y)[at] = static_cast<_Float16>(s);
}

// 4-bit quantiser: per group of 32, 64 or 128 columns of a row
//   without zero points  s = max |w| / 7 rounded to its type,             q = clamp(round(w / s) + 8, 0, 15)
//   with them            s = (max(w, 0) - min(w, 0)) / 15 rounded,        z = round(-min(w, 0) / s),  q = clamp(round(w / s) + z, 0, 15)
// A group of zeros has s = 0 and q = 8 (z = 0, q = 0 with zero points); so has one whose s rounds to 0.  A group that holds a NaN or an
// infinity, or whose range fp32 does not hold, has s = NaN: minima and maxima pass NaN over, and its codes would be those of ordinary
// weights.  8 columns a lane, one store of 4 bytes.
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
  return static_cast<float>(static_cast<_Float16>(v));
}

// A group's lanes hold eight columns each.  Run once per weight: 4096 x 7168 29 us, 2.6 TB/s, with a division for each weight, where one
// reciprocal a group would do.
template <int T>
__global__ void __launch_bounds__(256) w4_quant_kernel(const W4QuantArgs p) {
  const int lanes = p.group / 8;  // of a group: 4, 8 or 16
  const int64_t total = p.rows * p.G;
  const int sub = threadIdx.x % lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256 / lanes;
  for (int64_t g = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / lanes; g < total; g += step) {
    const int64_t row = g / p.G, kg = g - row * p.G;
    float v[8];
    quant_unpack8<T>(load_raw8<T, true>(p.w, row * p.w_rs, static_cast<int>(kg * p.group) + 8 * sub, 8), v);
    float hi = 0.f, lo = 0.f;
    uint32_t top = 0;  // the largest magnitude as bits, which put infinity above all numbers and NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) hi = fmaxf(hi, v[i]), lo = fminf(lo, v[i]), top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    for (int off = lanes / 2; off >= 1; off >>= 1) {
      hi = fmaxf(hi, __shfl_xor(hi, off, lanes)), lo = fminf(lo, __shfl_xor(lo, off, lanes));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, lanes)));
    }
    const float range = p.z ? hi - lo : fmaxf(hi, -lo);
    constexpr uint32_t kInf = 0x7f800000u;
    const bool numbers = top < kInf && __float_as_uint(fabsf(range)) < kInf;
    const float s = numbers ? round_to_type<T>(range / (p.z ? 15.0f : 7.0f)) : __uint_as_float(0x7fc00000u);
    const float zero = p.z ? (s > 0.f ? fminf(rintf(-lo / s), 15.f) : 0.f) : 8.f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = s > 0.f ? fminf(fmaxf(rintf(v[i] / s) + zero, 0.f), 15.f) : zero;
      word |= static_cast<uint32_t>(c) << (4 * i);
    }
    reinterpret_cast<uint32_t*>(p.q)[g * lanes + sub] = word;
    if (sub == 0) {
      if (T == kInBf16)
        static_cast<__bf16*>(p.s)[g] = static_cast<__bf16>(s);
      else
        static_cast<_Float16*>(p.s)[g] = static_cast<_Float16>(s);
      if (p.z) p.z[g] = static_cast<uint8_t>(zero);
    }
  }
}

}  // namespace dlb
