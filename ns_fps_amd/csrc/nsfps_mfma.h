// Matrix products of the selective scan on the matrix cores: 16 x 16 tiles of
// float32 sums over 32 terms at a time.
//
// One layout convention for everything, with g = lane / 16, l = lane % 16:
//   operand A holds row l, operand B column l, of terms k = 4g .. 4g+3 and
//   16 + 4g .. 16 + 4g+3 (two "quads" of four values);
//   the sum tile holds column l, rows 4g .. 4g+3.
// The order of the terms is the same in A and B, so it is free; this one makes
// the tile of a first product, as it lies in the registers, a quad of the
// operand B of a second one (its rows become the terms), with no exchange
// between lanes.  bfloat16: one 16x16x32 instruction; float32: eight 16x16x4,
// each taking one value of a quad.
#pragma once

#include "nsfps_seq_device.h"

#pragma clang fp contract(fast)

namespace nsfps {
namespace seq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// Four values of an operand; the element type of LDS tiles.
template <typename T>
struct QuadOf;
template <>
struct QuadOf<float> {
  typedef f32x4 type;
};
template <>
struct QuadOf<bf16> {
  typedef bf16x4 type;
};
template <typename T>
using Quad = typename QuadOf<T>::type;

// sum += A B over 32 terms
__device__ __forceinline__ void mma(f32x4 &sum, f32x4 a0, f32x4 a1, f32x4 b0, f32x4 b1) {
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[i], b0[i], sum, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[i], b1[i], sum, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4 &sum, bf16x4 a0, bf16x4 a1, bf16x4 b0, bf16x4 b1) {
  const bf16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
  const bf16x8 b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, sum, 0, 0, 0);
}


// The same with the products summed apart and added to sum by the vector
// unit.  The matrix unit aligns its addends and drops what falls below: a
// bfloat16 product added to a sum already there is off by 0.04 of 2^-24 of it
// on average, always downwards (16x16x32 on random values; 0.002 when the sum
// starts at zero, none in float32).  Summed over 10^5 tokens into a
// parameter's gradient, that shows.
__device__ __forceinline__ void mma_apart(f32x4 &sum, f32x4 a0, f32x4 a1, f32x4 b0, f32x4 b1) {
  mma(sum, a0, a1, b0, b1);
}
__device__ __forceinline__ void mma_apart(f32x4 &sum, bf16x4 a0, bf16x4 a1, bf16x4 b0, bf16x4 b1) {
  f32x4 z = {0.f, 0.f, 0.f, 0.f};
  mma(z, a0, a1, b0, b1);
  sum += z;
}

__device__ __forceinline__ f32x4 quad_f32(f32x4 q) { return q; }
__device__ __forceinline__ f32x4 quad_f32(bf16x4 q) { return __builtin_convertvector(q, f32x4); }

// A float32 value as operand terms whose sum it is: in bfloat16 one term keeps
// 8 bits, two 16, three all 24; in float32 one term is the value.  (Terms of
// magnitude below 2^-126 are lost; infinities do not split.)
template <typename T, int N>
struct Terms {
  static constexpr int kN = sizeof(T) == 4 ? 1 : N;
  Quad<T> q[kN];
};
template <typename T, int N>
__device__ __forceinline__ Terms<T, N> split(f32x4 v) {
  Terms<T, N> t;
  if constexpr (sizeof(T) == 4) {
    t.q[0] = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      t.q[i] = __builtin_convertvector(v, bf16x4);
      if (i + 1 < N) v -= quad_f32(t.q[i]);
    }
  }
  return t;
}

// LDS tiles: rows of `ld` elements, padded by 16 bytes so that the 16 rows a
// quarter of a wave reads at once start in different banks.
template <typename T, int COLS>
constexpr int kLd = COLS + 16 / (int)sizeof(T);

// terms along the row: row r, terms k .. k+3
template <typename T>
__device__ __forceinline__ Quad<T> quad_row(const T *tile, int ld, int r, int k) {
  return *(const Quad<T> *)(tile + r * ld + k);
}
// terms down the column: column c, terms (rows) k .. k+3
template <typename T>
__device__ __forceinline__ Quad<T> quad_col(const T *tile, int ld, int k, int c) {
  Quad<T> q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4)
      q[i] = tile[(k + i) * ld + c];
    else
      q[i] = __builtin_bit_cast(__bf16, tile[(k + i) * ld + c].u);
  }
  return q;
}

// A tile of 64 rows x COLS columns from global rows, zeros from row `rows` and
// column `cols` on; 256 threads.  wide: rows start at 16-byte boundaries and
// cols is a multiple of the elements in 16 bytes.
template <typename T, int COLS>
__device__ __forceinline__ void load_tile(T *tile, const T *g, uint64_t row_stride, uint32_t rows,
                                          uint32_t cols, bool wide) {
  constexpr int V = kWide<T>, kVecs = COLS / V, ld = kLd<T, COLS>;
  if (wide) {
#pragma unroll
    for (uint32_t e = threadIdx.x; e < 64 * kVecs; e += 256) {
      const uint32_t r = e / kVecs, c = (e % kVecs) * V;
      u32x4 v = {0, 0, 0, 0};
      if (r < rows && c < cols)
        v = *(const NSFPS_GLOBAL_SEQ u32x4 *)(g + r * row_stride + c);
      *(u32x4 *)(tile + r * ld + c) = v;
    }
  } else {
    for (uint32_t e = threadIdx.x; e < 64 * COLS; e += 256) {
      const uint32_t r = e / COLS, c = e % COLS;
      float v[1] = {0.f};
      if (r < rows && c < cols) load_f32<T, 1>(g + r * row_stride + c, v);
      tile[r * ld + c] = from_f32<T>(v[0]);
    }
  }
}

}  // namespace seq
}  // namespace nsfps
