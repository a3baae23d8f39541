// Tokens sorted by expert and back, with their gradients, for gfx950.
//
//   slots      (t, j) with 0 <= ids[t, j] < E, ordered by (expert, t, j): a stable counting sort, the same in every run
//   spans      expert e owns rows [start_e, end_e), start_e = sum over the experts before of their counts rounded up to `align`;
//              what would lie at or past the last reserved row is dropped
//   permute    rows[row_index[t, j]] = x[t], all other rows zero
//   unpermute  out[t] = sum_j w[t, j] rows[row_index[t, j]] over the slots with a row, an fp32 FMA chain in slot order
//   gradients  of permute: unpermute without weights.  Of unpermute: drows[row] = w dout[t] (zero in rows without a slot),
//              dw[t, j] = sum over the columns of rows[row] dout[t]
//
// ep_scatter and ep_gather (moe_permute.h) are the forms for spans that a dispatcher has already sized on the host; here the
// counts are found on the device and the rows carry gradients.  Copies and sums are bound by memory: a token's chunk is held in
// registers while all of its rows are written or read, so either side is touched once.
#pragma once

#include "fp8_gemm_common.h"
#include "rms_norm.h"

namespace dlb {

constexpr int kSortMaxTopk = 64;
constexpr int kSortThreads = 1024;
constexpr int kSortBlockSlots = 1024;     // slots whose rows one workgroup of the table kernel finds
constexpr int kSortMaxExperts = 1024;  // tables of the workgroups in 64 KB of LDS

struct SortArgs {
  const void* ids;      // [T][topk], < 0 or >= E: no expert
  int32_t* row_index;   // [T * topk]: row of every slot, -1: none
  int32_t* source;      // [R]: slot of every row, -1: none
  int32_t* m_indices;   // [R]: expert of every row of a span, -1 past the last span
  int32_t* row_start;   // [E]
  int32_t* row_end;     // [E]: one past the last row with a slot
  int32_t* hist;        // [blocks][E], used by launches of more than one workgroup of slots; summed: [blocks + 1][E], slots before
  int64_t ids_s0, ids_s1;
  int64_t n;            // T * topk
  int64_t R;
  int ids_is64, E, topk, align;
};

__device__ __forceinline__ int sort_id(const SortArgs& p, int64_t i) {
  if (i >= p.n) return -1;
  const int64_t t = static_cast<uint32_t>(i) / static_cast<uint32_t>(p.topk);  // n fits the int32 tables
  const int64_t at = t * p.ids_s0 + (i - t * p.topk) * p.ids_s1;
  const int64_t id = p.ids_is64 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<int64_t>(static_cast<const int32_t*>(p.ids)[at]);
  return (id < 0 || id >= p.E) ? -1 : static_cast<int>(id);
}

// Slots of every expert among the workgroup's 1024: 32768 slots 4.7 us, launch and latency.
__global__ void __launch_bounds__(kSortThreads) moe_sort_count_kernel(const SortArgs p) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e < p.E; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const int id = sort_id(p, static_cast<int64_t>(blockIdx.x) * kSortBlockSlots + threadIdx.x);
  if (id >= 0) atomicAdd(&hist[id], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kSortThreads) p.hist[static_cast<int64_t>(blockIdx.x) * p.E + e] = hist[e];
}

// Rows moved as bytes in chunks of 16; the last chunk of a row may be short (not where rows are WHOLE chunks).
template <bool WHOLE>
__device__ __forceinline__ v4i load_bytes16(const char* p, int left, int esz) {
  if (WHOLE || left >= 16) return *reinterpret_cast<const v4i_el*>(p);
  v4i v{0, 0, 0, 0};
  if (esz == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (2 * i < left) v[i / 2] |= static_cast<int>(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1)));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * i < left) v[i] = reinterpret_cast<const int*>(p)[i];
  }
  return v;
}
template <bool WHOLE>
__device__ __forceinline__ void store_bytes16(char* p, const v4i& v, int left, int esz) {
  if (WHOLE || left >= 16) {
    *reinterpret_cast<v4i_el*>(p) = v;
  } else if (esz == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (2 * i < left) reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(static_cast<uint32_t>(v[i / 2]) >> (16 * (i & 1)));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * i < left) reinterpret_cast<int*>(p)[i] = v[i];
  }
}

struct SortCopyArgs {
  const char* x;        // [T] rows of row_bytes
  char* rows;           // [R]
  const float* xs;      // scales of quantised tokens [T][groups] or NULL
  float* rows_s;        // [R][groups]
  const int32_t* row_index;
  const int32_t* source;
  int64_t x_stride, rows_stride;  // bytes
  int64_t xs_s0, xs_s1;
  int64_t T, R;
  int row_bytes, esz, topk, groups;
  int parts, part_bytes;          // a token's row is cut into parts, a wave's work each
  int token_blocks, zero_blocks;
};

constexpr int kSortCopyThreads = 256;
constexpr int kSortCopyChunks = 4;  // of 16 bytes a lane holds while a token's rows are written

// Part `part` of token t to all of its rows by one wave, lane j holding the row of slot j (-1: none).  A token without a row is not read.
template <bool WHOLE>
__device__ __forceinline__ void copy_token(const SortCopyArgs& p, int64_t t, int part, int mine, int lane) {
  const uint64_t there = __ballot(mine >= 0);
  if (there == 0) return;
  const char* src = p.x + t * p.x_stride;
  const int end = min(p.row_bytes, (part + 1) * p.part_bytes);
  for (int c0 = part * p.part_bytes; c0 < end; c0 += kSortCopyChunks * 1024) {
    v4i v[kSortCopyChunks];
#pragma unroll
    for (int k = 0; k < kSortCopyChunks; ++k) {
      const int c = c0 + (k * 64 + lane) * 16;
      if (c < end) v[k] = load_bytes16<WHOLE>(src + c, p.row_bytes - c, p.esz);
    }
    for (uint64_t left = there; left; left &= left - 1) {
      char* dst = p.rows + static_cast<int64_t>(__builtin_amdgcn_readlane(mine, __builtin_ctzll(left))) * p.rows_stride;
#pragma unroll
      for (int k = 0; k < kSortCopyChunks; ++k) {
        const int c = c0 + (k * 64 + lane) * 16;
        if (c < end) store_bytes16<WHOLE>(dst + c, v[k], p.row_bytes - c, p.esz);
      }
    }
  }
  if (part != 0) return;
  for (int g0 = 0; g0 < p.groups; g0 += 64) {
    const int g = g0 + lane;
    const float s = g < p.groups ? p.xs[t * p.xs_s0 + g * p.xs_s1] : 0.f;
    for (uint64_t left = there; left; left &= left - 1) {
      const int64_t row = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
      if (g < p.groups) p.rows_s[row * p.groups + g] = s;
    }
  }
}

template <bool WHOLE>
__device__ __forceinline__ void clear_row(const SortCopyArgs& p, int64_t r, int lane) {
  char* dst = p.rows + r * p.rows_stride;
  for (int c = lane * 16; c < p.row_bytes; c += 64 * 16) store_bytes16<WHOLE>(dst + c, v4i{0, 0, 0, 0}, p.row_bytes - c, p.esz);
  for (int g = lane; g < p.groups; g += 64) p.rows_s[r * p.groups + g] = 0.f;
}

// Counts to slots in the workgroups before, the totals in a row of their own.  A lane an expert, the waves take stretches of the
// workgroups of slots: their sums first, then again from the sums of the waves before.  516 workgroups, 256 experts 7.1 us, 7813 69 (one
// wave for all of them 26 and 372).
constexpr int kScanWaves = 16;

__global__ void __launch_bounds__(64 * kScanWaves) moe_sort_scan_kernel(const SortArgs p, int slot_blocks) {
  __shared__ int sums[kScanWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e = blockIdx.x * 64 + lane;
  int32_t* const hist = p.hist + min(e, p.E - 1);
  const int each = (slot_blocks + kScanWaves - 1) / kScanWaves;
  const int first = min(wave * each, slot_blocks), last = min(first + each, slot_blocks);
  const auto counts = [&](int b, int (&c)[8]) {
#pragma unroll
    for (int u = 0; u < 8; ++u) c[u] = hist[static_cast<int64_t>(min(b + u, slot_blocks - 1)) * p.E];
  };
  int sum = 0;
  for (int b = first; b < last; b += 8) {
    int c[8];
    counts(b, c);
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += b + u < last ? c[u] : 0;
  }
  sums[wave][lane] = sum;
  __syncthreads();
  sum = 0;
  for (int w = 0; w < wave; ++w) sum += sums[w][lane];
  if (e >= p.E) return;
  for (int b = first; b < last; b += 8) {
    int c[8];
    counts(b, c);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (b + u >= last) break;
      hist[static_cast<int64_t>(b + u) * p.E] = sum;
      sum += c[u];
    }
  }
  if (wave == kScanWaves - 1) hist[static_cast<int64_t>(slot_blocks) * p.E] = sum;
}

// Rows of the slots of workgroup blockIdx, and its share of the tables by row.  Workgroups past the slots' share only the latter.
// COPY: there is one workgroup's worth of slots, and every workgroup finds the rows of all of them and copies its share of the tokens, so
// that a few tokens take one launch.  Then only the first workgroup writes the tables by slot and expert.
// 32768 slots 5.8 us and 4.7 for the counts before it, both latency: loads, LDS atomics, barriers.
// LDS: before [E], total [E], start [E + 1], wave_cnt [16][E] of 16-bit counts; COPY: rows [threads].
template <bool COPY, bool WHOLE>
__global__ void __launch_bounds__(kSortThreads) moe_sort_rows_kernel(const SortArgs p, int slot_blocks, bool summed, const SortCopyArgs c) {
  extern __shared__ int lds[];
  const int E = p.E;
  int* before = lds;           // slots of the expert in the workgroups before, then the expert's next row in this one
  int* total = before + E;     // slots of the expert
  int* start = total + E;      // [E + 1] first row of every span
  uint16_t* wave_cnt = reinterpret_cast<uint16_t*>(start + E + 1);  // [16][E]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), threads = blockDim.x;
  const int b = blockIdx.x;
  const bool slots_here = COPY || b < slot_blocks;
  int* const rows = reinterpret_cast<int*>(wave_cnt + 16 * E);  // an even number of them before
  for (int i = tid; i < 2 * E; i += threads) lds[i] = 0;
  for (int i = tid; i < 16 * E; i += threads) wave_cnt[i] = 0;
  __syncthreads();
  const int64_t slot = COPY ? tid : static_cast<int64_t>(b) * kSortBlockSlots + tid;
  const int id = slots_here ? sort_id(p, slot) : -1;
  if (slot_blocks == 1) {
    // one workgroup of slots: every workgroup counts them itself
    const int mine = COPY || b == 0 ? id : sort_id(p, tid);
    if (mine >= 0) atomicAdd(&total[mine], 1);
  } else if (summed) {
    for (int e = tid; e < E; e += threads) {
      total[e] = p.hist[static_cast<int64_t>(slot_blocks) * E + e];
      before[e] = b < slot_blocks ? p.hist[static_cast<int64_t>(b) * E + e] : 0;
    }
  } else {
    const int cols = min(E, kSortThreads), P = kSortThreads / cols;
    const int my_part = tid / cols, my_col = tid % cols;
    for (int e = my_col; e < E && my_part < P; e += cols) {
      int all = 0, early = 0;
      for (int r = my_part; r < slot_blocks; r += P) {
        const int c = p.hist[static_cast<int64_t>(r) * E + e];
        all += c;
        if (r < b) early += c;
      }
      if (all) atomicAdd(&total[e], all);
      if (early) atomicAdd(&before[e], early);
    }
  }
  __syncthreads();
  if (wave == 0) {
    int64_t carry = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      const int e = e0 + lane;
      const int64_t c = e < E ? (static_cast<int64_t>(total[e]) + p.align - 1) / p.align * p.align : 0;
      int64_t incl = c;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int64_t up = __shfl_up(incl, off);
        if (lane >= off) incl += up;
      }
      if (e < E) start[e] = static_cast<int>(min(carry + incl - c, p.R));
      carry += __shfl(incl, 63);
    }
    if (lane == 0) start[E] = static_cast<int>(min(carry, p.R));
  }
  // slots with the same expert: in the waves before (wave_cnt) and in the lanes before (one ballot per bit of the id)
  uint64_t same = ~0ull;
  if (slots_here) {
    const uint64_t live = __ballot(id >= 0);
    same = live;
    for (int bit = 0; (E - 1) >> bit; ++bit) {
      const uint64_t ones = __ballot((id >> bit) & 1);
      same &= ((id >> bit) & 1) ? ones : ~ones;
    }
    if (id >= 0 && (same >> lane) == 1) wave_cnt[wave * E + id] = static_cast<uint16_t>(__popcll(same));
  }
  __syncthreads();
  if (slots_here && slot < p.n) {
    int64_t row = -1;
    if (id >= 0) {
      row = static_cast<int64_t>(start[id]) + before[id] + __popcll(same & ((1ull << lane) - 1));
      for (int w = 0; w < wave; ++w) row += wave_cnt[w * E + id];
      if (row >= p.R) row = -1;
    }
    if (COPY) rows[tid] = static_cast<int>(row);
    if (!COPY || b == 0) {
      p.row_index[slot] = static_cast<int32_t>(row);
      if (row >= 0) p.source[row] = static_cast<int32_t>(slot);
    }
  }
  if (b == 0)
    for (int e = tid; e < E; e += threads) {
      p.row_start[e] = start[e];
      p.row_end[e] = static_cast<int>(min(static_cast<int64_t>(start[e]) + total[e], p.R));
    }
  const auto expert_of = [&](int64_t r) {  // of row r, -1: past the last span
    if (r >= start[E]) return -1;
    int lo = 0, hi = E;  // the last e with start[e] <= r: an empty span before it starts at the same row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  };
  const auto vacant = [&](int64_t r, int e) { return e < 0 || r >= static_cast<int64_t>(start[e]) + total[e]; };
  for (int64_t r = static_cast<int64_t>(b) * threads + tid; r < p.R; r += static_cast<int64_t>(gridDim.x) * threads) {
    const int e = expert_of(r);
    p.m_indices[r] = e;
    if (vacant(r, e)) p.source[r] = -1;
  }
  if (!COPY) return;
  __syncthreads();
  const int waves = threads / 64;
  for (uint32_t u = b * waves + wave; u < static_cast<uint32_t>(c.T * c.parts); u += gridDim.x * waves) {  // at most 1024 parts of 2^20 KB
    const int t = static_cast<int>(u / static_cast<uint32_t>(c.parts));
    copy_token<WHOLE>(c, t, static_cast<int>(u) - t * c.parts, lane < p.topk ? rows[t * p.topk + lane] : -1, lane);
  }
  for (int64_t r = static_cast<int64_t>(b) * waves + wave; r < p.R; r += static_cast<int64_t>(gridDim.x) * waves)
    if (vacant(r, expert_of(r))) clear_row<WHOLE>(c, r, lane);
}

// A wave per token and part: blocks [0, token_blocks) take the tokens, the others look for rows without a slot.  The slots' rows come
// in one load, a lane each.  Few tokens are cut finer, so that there are waves for the whole chip.  4096 x 7168 bf16 to 8 rows each, 528 MB:
// 93 us (5.7 TB/s), 8192 x 7168 e4m3 with one in eight of
// 8 slots here, 167 MB, 26.
template <bool WHOLE>
__global__ void __launch_bounds__(kSortCopyThreads) moe_sort_copy_kernel(const SortCopyArgs p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kWaves = kSortCopyThreads / 64;
  if (static_cast<int>(blockIdx.x) < p.token_blocks) {
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWaves + wave; u < p.T * p.parts; u += static_cast<int64_t>(p.token_blocks) * kWaves) {
      const int64_t t = u / p.parts;
      copy_token<WHOLE>(p, t, static_cast<int>(u - t * p.parts), lane < p.topk ? p.row_index[t * p.topk + lane] : -1, lane);
    }
    return;
  }
  const int64_t zb = static_cast<int64_t>(blockIdx.x) - p.token_blocks;
  for (int64_t r = zb * kWaves + wave; r < p.R; r += static_cast<int64_t>(p.zero_blocks) * kWaves)
    if (p.source[r] < 0) clear_row<WHOLE>(p, r, lane);
}

struct UnpermuteArgs {
  const void* rows;         // [R][H]
  const int32_t* row_index; // [T][topk]
  const float* w;           // [T][topk] or NULL: all one
  void* out;                // [T][H]
  int64_t rows_rs, out_rs;  // elements
  int64_t T, R;
  int H, topk;
};

// One wave per token and stretch of 512 columns (a chunk a lane); the slots' rows and weights come in one load each, a lane a slot.  The
// chunks of kUnpermuteRows rows are on their way at a time, behind the last row that one again.  4096 tokens x 8 rows of 7168 bf16, 528 MB:
// 131 us, 4.0 TB/s (streams in order reach 6.0 here, with the non-temporal bit 7.0; these loads do not have it); the stretches of a token next
// to each other in the grid, or two and seven of them by one wave, took 133, 130 and 130.  1001 x 4096, two thirds of 6 slots here: 8.9 us.
constexpr int kUnpermuteRows = 4;

template <int T, bool WHOLE>
__global__ void __launch_bounds__(64) moe_unpermute_kernel(const UnpermuteArgs p) {
  const int lane = threadIdx.x;
  const int64_t t = static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x;
  if (t >= p.T) return;
  int mine = lane < p.topk ? p.row_index[t * p.topk + lane] : -1;
  if (mine >= p.R) mine = -1;
  const float my_w = lane < p.topk && p.w ? p.w[t * p.topk + lane] : 1.f;
  const uint64_t there = __ballot(mine >= 0);
  const int chunks = (p.H + 7) / 8;
  for (int c0 = blockIdx.y * 64; c0 < chunks; c0 += gridDim.y * 64) {
    const int col = min(c0 + lane, chunks - 1) * 8, left = p.H - col;
    float acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
    for (uint64_t todo = there; todo;) {
      Raw8 raw[kUnpermuteRows];
      float wj[kUnpermuteRows];
      const int n = __popcll(todo);
      int j = 0;
#pragma unroll
      for (int u = 0; u < kUnpermuteRows; ++u) {
        if (todo) j = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int64_t row = __builtin_amdgcn_readlane(mine, j);
        wj[u] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_w), j));
        raw[u] = load_raw8<T, WHOLE>(p.rows, row * p.rows_rs, col, left);
      }
#pragma unroll
      for (int u = 0; u < kUnpermuteRows; ++u) {
        if (u >= n) break;
        float v[8];
        quant_unpack8<T>(raw[u], v);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = fmaf(v[k], wj[u], acc[k]);
      }
    }
    if (c0 + lane < chunks) store_raw8<T, WHOLE>(p.out, t * p.out_rs, col, pack_raw8<T>(acc), left);
  }
}

struct UnpermuteGradArgs {
  const void* dout;         // [T][H]
  const void* rows;         // [R][H], read for dw only
  const int32_t* row_index;
  const int32_t* source;    // [R]
  const float* w;           // [T][topk] or NULL: all one
  void* drows;              // [R][H]
  float* dw;                // [T][topk] or NULL
  int64_t dout_rs, rows_rs, drows_rs;
  int64_t T, R;
  int H, topk;
  int zero_blocks;
};

// One workgroup per token, the chunks of its gradient in registers (CH a thread) while its rows pass; the workgroups behind the
// tokens write the rows without a slot.  The waves' shares of a slot's product meet in LDS.  DW: with the gradient of the weights, the
// only reader of the rows; those of kAhead slots are on their way at a time, for a slot without a row the first one in its place.
// 4096 tokens x 8 rows of 7168 bf16, 1.0 GB: 195 us, 5.1 TB/s.
template <int T, bool DW, bool WHOLE, int CH>
__global__ void __launch_bounds__(kNormMaxThreads) moe_unpermute_backward_kernel(const UnpermuteGradArgs p) {
  __shared__ float part[kSortMaxTopk][kNormMaxWaves];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int chunks = (p.H + 7) / 8;
  const int64_t t = grid_row();
  if (t >= p.T) {
    Raw8 zero;
    zero.a = v4i{0, 0, 0, 0}, zero.b = v4i{0, 0, 0, 0};
    for (int64_t r = t - p.T; r < p.R && t < p.T + p.zero_blocks; r += p.zero_blocks) {
      if (p.source[r] >= 0) continue;
      for (int i = tid; i < chunks; i += threads) store_raw8<T, WHOLE>(p.drows, r * p.drows_rs, 8 * i, zero, p.H - 8 * i);
    }
    return;
  }
  if (p.R == 0) {
    if (DW && tid < p.topk) p.dw[t * p.topk + tid] = 0.f;
    return;
  }
  const int32_t* index = p.row_index + t * p.topk;
  const float* w = p.w ? p.w + t * p.topk : nullptr;
  int at[CH];
  Raw8 g[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    at[c] = min(c * threads + tid, chunks - 1);
    g[c] = load_raw8<T, WHOLE>(p.dout, t * p.dout_rs, 8 * at[c], p.H - 8 * at[c]);
  }
  constexpr int kAhead = CH == 1 ? 4 : 2;
  for (int j0 = 0; j0 < p.topk; j0 += kAhead) {
    Raw8 raw[kAhead][CH];
    int64_t row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      row[u] = j0 + u < p.topk ? index[j0 + u] : -1;
      if (row[u] >= p.R) row[u] = -1;
      if (!DW) continue;
#pragma unroll
      for (int c = 0; c < CH; ++c) raw[u][c] = load_raw8<T, WHOLE>(p.rows, max(row[u], int64_t{0}) * p.rows_rs, 8 * at[c], p.H - 8 * at[c]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j0 + u >= p.topk) break;
      float dot = 0.f;
      if (row[u] >= 0) {
        const float wj = w ? w[j0 + u] : 1.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          if (c * threads + tid >= chunks) continue;
          float d[8];
          quant_unpack8<T>(g[c], d);
          if (DW) {
            float v[8];
            quant_unpack8<T>(raw[u][c], v);
#pragma unroll
            for (int k = 0; k < 8; ++k) dot = fmaf(v[k], d[k], dot);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) d[k] *= wj;
          store_raw8<T, WHOLE>(p.drows, row[u] * p.drows_rs, 8 * at[c], pack_raw8<T>(d), p.H - 8 * at[c]);
        }
      }
      if (DW) {
        dot = wave_sum(dot);
        if ((tid & 63) == 0) part[j0 + u][tid >> 6] = dot;
      }
    }
  }
  if (!DW) return;
  __syncthreads();
  for (int j = tid; j < p.topk; j += threads) {
    float s = 0.f;
    for (int i = 0; i < threads / 64; ++i) s += part[j][i];
    p.dw[t * p.topk + j] = s;
  }
}

}  // namespace dlb
