// Products of bfloat16 matrices on the matrix cores, fed straight from global
// memory to LDS: a workgroup's tile of sums C[m][n] = sum over k of M[m][k] N[n][k].
//
// An operand lies in memory with its terms k along the row (Row: element (m, k)
// at m * ld + k) or down the column (Col: at k * ld + m).  Stages of 64 terms go
// to LDS in 16-byte pieces, 64 of them an instruction in the order of the lanes,
// so a tile's rows have no padding; the pieces of a row are exchanged instead,
// by a number that the row gives, so that the 16 rows which lanes read at once
// lie in different banks.  Reads of a Col tile transpose on the way.
//
// Lane layout, with g = lane / 16, l = lane % 16: an operand of 32 terms holds
// row l, terms 8g .. 8g + 7; a tile of sums holds row m = l, columns n = 4g .. 4g
// + 3.  kPerm (four column tiles): column 4g + r of tile nt stands for column 16g
// + 4nt + r of the wave's 64, so that a lane's 16 sums of a row are neighbours.
//
// Sizes are whole: tiles inside the operands, terms a multiple of 64.
#pragma once

#include "nsfps_mfma.h"

#pragma clang fp contract(fast)

namespace nsfps {
namespace seq {

constexpr uint32_t kStage = 64;  // terms of a stage

// The number that exchanges a row's pieces.  Row: 128 bytes a row, 8 pieces; the
// rows 0 .. 15 and the rows 16a + 4c + b (a, b < 4) get all 8 at both parities.
__device__ __forceinline__ uint32_t row_turn(uint32_t r) {
  return ((r >> 1) & 1) | ((((r >> 2) + (r >> 4)) & 3) << 1);
}
// Col: pairs of pieces (16 columns); rows 8g + i (g, i < 4).
template <int T>
__device__ __forceinline__ uint32_t col_turn(uint32_t k) {
  if constexpr (T == 64) return (((k >> 1) & 1) | ((k >> 2) & 2)) << 1;
  return ((k & 3) | ((k >> 1) & 4)) << 1;
}

// The pieces of an operand's stage that this thread brings.
template <int T, bool kCol, int kThreads>
struct Feed {
  static constexpr int kPer = T * (int)kStage / 8 / kThreads;
  static_assert(kPer >= 1, "tile too small");
  const bf16 *p[kPer];

  // at: the tile's first row (Row) or column (Col) at term 0
  __device__ __forceinline__ void start(const bf16 *at, uint64_t ld) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + kThreads * i;
      if constexpr (kCol) {
        const uint32_t k = e / (T / 8), c = (e % (T / 8)) ^ col_turn<T>(k);
        p[i] = at + k * ld + 8 * c;
      } else {
        const uint32_t r = e / 8, c = (e % 8) ^ row_turn(r);
        p[i] = at + r * ld + 8 * c;
      }
    }
  }
  __device__ __forceinline__ void issue(bf16 *stage, uint64_t offset) const {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void *)(p[i] + offset),
          (__attribute__((address_space(3))) void *)(stage + 8 * (64 * wave + kThreads * i)), 16, 0,
          0);
  }
};

// A lane's operand of terms 32 kb .. 32 kb + 31; r: this lane's row.
__device__ __forceinline__ bf16x8 read_row(const bf16 *stage, uint32_t r, uint32_t kb, uint32_t g) {
  return *(const bf16x8 *)(stage + 8 * (8 * r + ((4 * kb + g) ^ row_turn(r))));
}
// c: the tile's first column
template <int T>
__device__ __forceinline__ bf16x8 read_col(const bf16 *stage, uint32_t c, uint32_t kb, uint32_t g,
                                           uint32_t l) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const uint32_t k = 32 * kb + 8 * g + l / 4, at = c + 4 * (l % 4);
  bf16x4 q[2];
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t row = k + 4 * i;
    q[i] = __builtin_bit_cast(
        bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s16x4 *)(stage + row * T + 8 * ((at / 8) ^ col_turn<T>(row)) + at % 8)));
  }
  return __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7);
}

// WM x WN waves of MT x NT tiles of 16 x 16 sums.
template <int WM, int WN, int MT, int NT, bool kMCol, bool kNCol, bool kPerm>
struct Product {
  static constexpr int kM = 16 * WM * MT, kN = 16 * WN * NT, kThreads = 64 * WM * WN;
  static_assert(!kPerm || (NT == 4 && !kNCol), "layout");
  struct alignas(16) Lds {
    bf16 m[2][kM * kStage], n[2][kN * kStage];
  };
  Feed<kM, kMCol, kThreads> fm;
  Feed<kN, kNCol, kThreads> fn;

  __device__ __forceinline__ void issue(Lds &lds, uint32_t buf, uint64_t m, uint64_t n) const {
    fm.issue(lds.m[buf], m);
    fn.issue(lds.n[buf], n);
  }
  // Waits for the stage issued last, adds its products; next() issues the one
  // after it, once this one's operands are in registers: the other half of LDS
  // was read before the barrier.
  template <typename F>
  __device__ __forceinline__ void add(f32x4 (&sum)[MT][NT], const Lds &lds, uint32_t buf, F next) {
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m0 = wave / WN * (16 * MT), n0 = wave % WN * (16 * NT);
    wait_loads();
    __syncthreads();
    bf16x8 m[2][MT], n[2][NT];
#pragma unroll
    for (uint32_t kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
        m[kb][t] = kMCol ? read_col<kM>(lds.m[buf], m0 + 16 * t, kb, g, l)
                         : read_row(lds.m[buf], m0 + 16 * t + l, kb, g);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        n[kb][t] = kNCol ? read_col<kN>(lds.n[buf], n0 + 16 * t, kb, g, l)
                   : kPerm ? read_row(lds.n[buf], n0 + 16 * (l / 4) + 4 * t + l % 4, kb, g)
                           : read_row(lds.n[buf], n0 + 16 * t + l, kb, g);
    }
    next();
#pragma unroll
    for (uint32_t kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(n[kb][j], m[kb][i], sum[i][j], 0, 0, 0);
  }
};

}  // namespace seq
}  // namespace nsfps
