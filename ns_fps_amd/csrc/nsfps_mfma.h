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


// Waits for the sums of products.  At the end of every branch that holds
// products: the compiler's own waits are not complete across its joins (a
// product, the branch, and a reader of the sum at the branch's target came out
// next to each other, and the reader had the old value).
template <typename T>
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (sizeof(T) == 4)
    asm volatile("s_nop 7\n\ts_nop 1" ::: "memory");  // 16x16x4 f32: 10 states
  else
    asm volatile("s_nop 7" ::: "memory");  // 16x16x32 bf16: 8 states
  __builtin_amdgcn_sched_barrier(0);
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
__device__ __forceinline__ f32x4 quad_f32(bf16x4 q) {
  const u32x2 w = __builtin_bit_cast(u32x2, q);
  return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u),
               __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)};
}

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
// quarter of a wave reads at once start in different banks.  In bfloat16 the
// columns of every 32 are stored with a lane's two quads next to each other
// (column 16a + 4g + r at 8g + 4a + r), so that both come in one 16-byte read.
template <typename T, int COLS>
constexpr int kLd = COLS + 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ int column_at(int c) {
  return sizeof(T) == 4 ? c : (c & ~31) | ((c & 12) << 1) | ((c & 16) >> 2) | (c & 3);
}

// Both quads of an operand of 32 terms.
template <typename T>
struct Pair {
  Quad<T> q0, q1;
};
template <typename T>
__device__ __forceinline__ void mma(f32x4 &sum, const Pair<T> &a, const Pair<T> &b) {
  mma(sum, a.q0, a.q1, b.q0, b.q1);
}
template <typename T>
__device__ __forceinline__ void mma_apart(f32x4 &sum, const Pair<T> &a, const Pair<T> &b) {
  mma_apart(sum, a.q0, a.q1, b.q0, b.q1);
}

// terms along the row: row r, terms 32 kb + this lane's
__device__ __forceinline__ Pair<float> pair_row(const float *tile, int ld, int r, int kb, int g) {
  const float *at = tile + r * ld + 32 * kb + 4 * g;
  return Pair<float>{*(const f32x4 *)at, *(const f32x4 *)(at + 16)};
}
__device__ __forceinline__ Pair<bf16> pair_row(const bf16 *tile, int ld, int r, int kb, int g) {
  const bf16x8 v = *(const bf16x8 *)(tile + r * ld + 32 * kb + 8 * g);
  return Pair<bf16>{__builtin_shufflevector(v, v, 0, 1, 2, 3), __builtin_shufflevector(v, v, 4, 5, 6, 7)};
}
// one quad of a row: columns c .. c+3, c a multiple of four
template <typename T>
__device__ __forceinline__ Quad<T> quad_row(const T *tile, int ld, int r, int c) {
  return *(const Quad<T> *)(tile + r * ld + column_at<T>(c));
}
template <typename T>
__device__ __forceinline__ void put_quad(T *tile, int ld, int r, int c, Quad<T> q) {
  *(Quad<T> *)(tile + r * ld + column_at<T>(c)) = q;
}

// terms down the column: columns c .. c+15 (this lane's: c + l), terms (rows)
// k .. k+3 with k the lane's own (a multiple of four plus 4g).  bfloat16: the
// transposing LDS read, in which the 16 lanes of a quarter read four rows of
// 16 elements and each receives a column; the whole wave takes part.
__device__ __forceinline__ f32x4 quad_col(const float *tile, int ld, int k, int c, int l) {
  f32x4 q;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = tile[(k + i) * ld + c + l];
  return q;
}
__device__ __forceinline__ bf16x4 quad_col(const bf16 *tile, int ld, int k, int c, int l) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const bf16 *at = tile + (k + l / 4) * ld + (c & ~31) + 8 * (l % 4) + ((c & 16) >> 2);
  return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)at));
}
// terms 32 kb + this lane's, down the column
template <typename T>
__device__ __forceinline__ Pair<T> pair_col(const T *tile, int ld, int kb, int c, int g, int l) {
  return Pair<T>{quad_col(tile, ld, 32 * kb + 4 * g, c, l),
                 quad_col(tile, ld, 32 * kb + 16 + 4 * g, c, l)};
}

// A tile of 64 rows x COLS columns on its way from global memory to LDS, in
// the registers of 256 threads: fetched while the tile before it is worked on.
// Rows past `rows` and columns past `cols` (both at least 1) are read from the
// last inside it and become zeros on the way to LDS: a load that is left out
// would have to be waited for before the next one into its registers.
// kWideRows: rows start at 16-byte boundaries and cols is a multiple of the
// elements in 16 bytes.
template <typename T, int COLS, bool kWideRows>
struct Tile {
  static constexpr int V = kWide<T>, kVecs = COLS / V, kPer = 64 * kVecs / 256;
  static_assert(kPer >= 1, "tile too small");
  u32x4 v[kPer];
  uint32_t rows, cols;

  __device__ __forceinline__ void fetch(const T *g, uint64_t row_stride, uint32_t nrows,
                                        uint32_t ncols) {
    rows = nrows;
    cols = ncols;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + 256 * i, c = (e % kVecs) * V;
      const NSFPS_GLOBAL_SEQ T *at =
          (const NSFPS_GLOBAL_SEQ T *)(g + min(e / kVecs, rows - 1) * row_stride);
      if constexpr (kWideRows) {
        v[i] = *(const NSFPS_GLOBAL_SEQ u32x4 *)(at + min(c, cols - V));
      } else {
        v[i] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
          const uint32_t ck = min(c + k, cols - 1);
          if constexpr (sizeof(T) == 4)
            v[i][k] = *(const NSFPS_GLOBAL_SEQ uint32_t *)(at + ck);
          else
            v[i][k / 2] |= (uint32_t) * (const NSFPS_GLOBAL_SEQ uint16_t *)(at + ck) << (16 * (k % 2));
        }
      }
    }
  }
  __device__ __forceinline__ void put(T *tile) {
    if (rows < 64 || cols < COLS) {  // the same for all lanes; most tiles are full
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t e = threadIdx.x + 256 * i, c = (e % kVecs) * V;
        const bool in = e / kVecs < rows;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          if constexpr (sizeof(T) == 4) {
            v[i][k] = in && c + k < cols ? v[i][k] : 0u;
          } else {
            const uint32_t keep = (in && c + 2 * k < cols ? 0xffffu : 0u) |
                                  (in && c + 2 * k + 1 < cols ? 0xffff0000u : 0u);
            v[i][k] &= keep;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + 256 * i;
      const int r = e / kVecs, c = (e % kVecs) * V;
      if constexpr (sizeof(T) == 4) {
        *(u32x4 *)(tile + r * kLd<T, COLS> + c) = v[i];
      } else {
        *(u32x2 *)(tile + r * kLd<T, COLS> + column_at<T>(c)) = u32x2{v[i].x, v[i].y};
        *(u32x2 *)(tile + r * kLd<T, COLS> + column_at<T>(c + 4)) = u32x2{v[i].z, v[i].w};
      }
    }
  }
};

}  // namespace seq
}  // namespace nsfps
