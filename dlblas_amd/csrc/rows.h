// Rows in registers: eight consecutive elements of a row as a chunk, loads and stores at any element boundary and of a short last chunk, sums
// over the lanes of a row.  What the kernels share that read a row once and leave it from the registers.
#pragma once

#include "fp8_gemm_common.h"
#include "fp8_quant.h"

namespace dlb {

typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef v4h v4h_el __attribute__((aligned(2)));

// Where column `col` of the row at element `row` lies: the row's start is the same in every lane, which leaves 32 bits a lane to keep.
template <int T>
__device__ __forceinline__ const char* raw8_at(const void* p, int64_t row, int col) {
  constexpr int kBytes = T == kInF32 ? 4 : 2;
  return static_cast<const char*>(p) + row * kBytes + static_cast<uint32_t>(col) * kBytes;
}

// Eight consecutive elements of a row as they lie in memory (16 bytes, 32 of fp32); `left` (at least 1) = elements left in the row, those
// past it are zero.  WHOLE: rows are a multiple of eight wide and there is no such case, nor the branch for it: waits for loads count
// those issued since, and behind a branch the compiler takes the lower count, so that a row asked for ahead would be waited for at once.
template <int T, bool WHOLE = false>
__device__ __forceinline__ Raw8 load_raw8(const void* p, int64_t row, int col, int left) {
  Raw8 r;
  r.a = v4i{0, 0, 0, 0}, r.b = v4i{0, 0, 0, 0};
  if (T == kInF32) {
    typedef v4i v4i_f32 __attribute__((aligned(4)));
    const float* q = reinterpret_cast<const float*>(raw8_at<T>(p, row, col));
    if (WHOLE || left >= 8) {
      r.a = reinterpret_cast<const v4i_f32*>(q)[0], r.b = reinterpret_cast<const v4i_f32*>(q)[1];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < left) r.a[i] = __float_as_int(q[i]);
        if (4 + i < left) r.b[i] = __float_as_int(q[4 + i]);
      }
    }
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(raw8_at<T>(p, row, col));
    if (WHOLE || left >= 8) {
      r.a = *reinterpret_cast<const v4i_el*>(q);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) r.a[i / 2] |= static_cast<int>(static_cast<uint32_t>(q[i]) << (16 * (i & 1)));
    }
  }
  return r;
}

// Eight fp32 values rounded to nearest even into the type of the rows.
template <int T>
__device__ __forceinline__ Raw8 pack_raw8(const float (&v)[8]) {
  Raw8 r;
  if (T == kInF32) {
    r.a = v4i{__float_as_int(v[0]), __float_as_int(v[1]), __float_as_int(v[2]), __float_as_int(v[3])};
    r.b = v4i{__float_as_int(v[4]), __float_as_int(v[5]), __float_as_int(v[6]), __float_as_int(v[7])};
  } else if (T == kInBf16) {
    const v2i lo = __builtin_bit_cast(v2i, __builtin_convertvector(v4f{v[0], v[1], v[2], v[3]}, v4bf));
    const v2i hi = __builtin_bit_cast(v2i, __builtin_convertvector(v4f{v[4], v[5], v[6], v[7]}, v4bf));
    r.a = v4i{lo.x, lo.y, hi.x, hi.y};
    r.b = r.a;
  } else {
    const v2i lo = __builtin_bit_cast(v2i, __builtin_convertvector(v4f{v[0], v[1], v[2], v[3]}, v4h));
    const v2i hi = __builtin_bit_cast(v2i, __builtin_convertvector(v4f{v[4], v[5], v[6], v[7]}, v4h));
    r.a = v4i{lo.x, lo.y, hi.x, hi.y};
    r.b = r.a;
  }
  return r;
}

template <int T, bool WHOLE = false>
__device__ __forceinline__ void store_raw8(void* p, int64_t row, int col, const Raw8& r, int left) {
  if (T == kInF32) {
    typedef v4i v4i_f32 __attribute__((aligned(4)));
    float* q = reinterpret_cast<float*>(const_cast<char*>(raw8_at<T>(p, row, col)));
    if (WHOLE || left >= 8) {
      reinterpret_cast<v4i_f32*>(q)[0] = r.a, reinterpret_cast<v4i_f32*>(q)[1] = r.b;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < left) q[i] = __int_as_float(r.a[i]);
        if (4 + i < left) q[4 + i] = __int_as_float(r.b[i]);
      }
    }
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(const_cast<char*>(raw8_at<T>(p, row, col)));
    if (WHOLE || left >= 8) {
      *reinterpret_cast<v4i_el*>(q) = r.a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) q[i] = static_cast<uint16_t>(static_cast<uint32_t>(r.a[i / 2]) >> (16 * (i & 1)));
    }
  }
}

// Over neighbouring LANES of a wave.
template <int LANES = 64>
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = LANES / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// The row, or the worker, of this thread among the blockDim.y beside each other in a workgroup: the same for a wave of one row.
template <int LANES>
__device__ __forceinline__ int beside() {
  return LANES < 64 ? static_cast<int>(threadIdx.y) : __builtin_amdgcn_readfirstlane(threadIdx.y);
}

// A barrier for what went through LDS; loads from memory stay on their way.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int T, bool WHOLE>
__device__ __forceinline__ void load_weight8(const void* w, int w_f32, int col, int left, float (&v)[8]) {
  if (w_f32)
    quant_unpack8<kInF32>(load_raw8<kInF32, WHOLE>(w, 0, col, left), v);
  else
    quant_unpack8<T>(load_raw8<T, WHOLE>(w, 0, col, left), v);
}

// A workgroup's place in a grid of two dimensions: one of them holds fewer than 2^32 threads.
__device__ __forceinline__ int64_t grid_row() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

}  // namespace dlb
