// Products of matrices on the matrix cores from tiles in LDS: a workgroup's tile
// of sums C[m][n] = sum over k of M[m][k] N[n][k], from operands whose terms lie
// along the row (Row: element (m, k) at m * ld + k) or down the column (Col: at
// k * ld + m) of memory.
//
// Operands in LDS are bfloat16; a float32 value is there as up to three terms
// whose sum it is, in planes, and its products are those of the planes that
// matter (Passes).  Rows of a tile have no padding; the 16-byte pieces of a row
// are exchanged instead, by a number that the row gives (the turn), so that rows
// which lanes read at once lie in different banks.  Reads of a Col tile transpose
// on the way.
//
// Tiles come to LDS in one of two ways: straight from memory where rows allow
// 16-byte pieces (Feed), or through registers from any rows of either type,
// which are split into planes and masked on the way (Stage).
//
// Lane layout, with g = lane / 16, l = lane % 16: an operand of 32 terms holds
// row l, terms 8g .. 8g + 7; a tile of sums holds row m = l, columns n = 4g .. 4g
// + 3.  kPerm: column 4g + r of the tiles 2t and 2t + 1 stands for columns 32t + 8g
// + r and + 4 + r, so that a lane has eight neighbours: 16 bytes of bfloat16.
#pragma once

#include "nsfps_mfma.h"

#pragma clang fp contract(fast)

namespace nsfps {
namespace seq {

// The number that exchanges the pieces of a row of kTerms terms (Row).  A 16-byte
// read takes 16 lanes at a time, rows 0 .. 3 and 12 .. 15 of one piece and rows 4
// .. 11 of the next one (then the other way round), over 256 bytes of banks.  One,
// two or four rows lie in those, so the others' bits have to give the piece, and
// with the pieces' own difference: by count no read meets a bank twice, be its rows 0 ..
// 15 or (kPerm) 8a + 4c + b (a, b < 4), and the hardware's counter of conflicts stays
// at 0 in every kernel of the loss.
template <int kTerms>
__device__ __forceinline__ uint32_t row_turn(uint32_t r) {
  static_assert(kTerms == 128 || kTerms == 64 || kTerms == 32, "terms of a stage");
  const uint32_t b3 = (r >> 3) & 1;
  return kTerms == 128 ? 9 * b3 | (r & 2) | (r & 1) << 2 : kTerms == 64 ? 5 * b3 | (r & 2) : 2 * b3;
}
// Col, T columns a row: pairs of pieces (16 columns); rows 8g + i (g, i < 4).
template <int T>
__device__ __forceinline__ uint32_t col_turn(uint32_t k) {
  if constexpr (T == 64) return (((k >> 1) & 1) | ((k >> 2) & 2)) << 1;
  return ((k & 3) | ((k >> 1) & 4)) << 1;
}

// Where the 8 values from column c (a multiple of 8) of memory row r go.
template <int T, int kTerms, bool kCol>
__device__ __forceinline__ uint32_t piece_at(uint32_t r, uint32_t c) {
  if constexpr (kCol) return r * T + 8 * ((c / 8) ^ col_turn<T>(r));
  return r * kTerms + 8 * ((c / 8) ^ row_turn<kTerms>(r));
}

// A lane's operand of terms 32 kb .. 32 kb + 31; r: this lane's row.
template <int kTerms>
__device__ __forceinline__ bf16x8 read_row(const bf16 *tile, uint32_t r, uint32_t kb, uint32_t g) {
  return *(const bf16x8 *)(tile + r * kTerms + 8 * ((4 * kb + g) ^ row_turn<kTerms>(r)));
}
// c: the first of the 16 columns
template <int T>
__device__ __forceinline__ bf16x8 read_col(const bf16 *tile, uint32_t c, uint32_t kb, uint32_t g,
                                           uint32_t l) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const uint32_t k = 32 * kb + 8 * g + l / 4, at = c + 4 * (l % 4);
  bf16x4 q[2];
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t row = k + 4 * i;
    q[i] = __builtin_bit_cast(
        bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s16x4 *)(tile + row * T + 8 * ((at / 8) ^ col_turn<T>(row)) + at % 8)));
  }
  return __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7);
}

// A tile straight from memory to LDS, 64 pieces of 16 bytes an instruction in
// the order of the lanes: the pieces' exchange is in the addresses.  Pieces are
// whole; memory rows past the last are the last one again.  Rows lie less than
// 2^23 values apart, so that a lane's place is a 32-bit offset from a base that
// all lanes share.
//
// The copies are written as instructions: the compiler, which takes every read of
// LDS behind such a copy for a read of what it brings, would wait for all of them
// there, and a tile could only be asked for once the one before it is in
// registers.  Nothing comes back to registers.  Whoever reads the tile waits
// himself: landed<n>() and a barrier.
template <int T, int kTerms, bool kCol, int kThreads>
struct Feed {
  static constexpr int kPer = T * kTerms / 8 / kThreads;  // copies a thread
  static_assert(kPer >= 1 && T * kTerms / 8 % kThreads == 0, "tile and threads");
  uint32_t at[kPer];  // bytes

  // rows: how many there are of memory from the tile's first on (at least 1)
  __device__ __forceinline__ void start(uint64_t ld, uint32_t rows) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + kThreads * i;
      constexpr uint32_t kVecs = kCol ? T / 8 : kTerms / 8;
      const uint32_t r = e / kVecs, turn = kCol ? col_turn<T>(r) : row_turn<kTerms>(r);
      at[i] = 2 * (min(r, rows - 1) * (uint32_t)ld + 8 * (e % kVecs ^ turn));
    }
  }
  // from: the tile's first value
  __device__ __forceinline__ void issue(bf16 *tile, const bf16 *from) const {
    const uint32_t to = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) bf16 *)tile +
        16 * (threadIdx.x & ~63u));
    const uint64_t base = (uint64_t)from;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      // (the compiler sets m0 itself, so that it knows what is there, but counts no
      // waits into these instructions: a scalar register that the vector unit wrote may
      // be read five states later, m0 one)
      asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
                   :
                   : "v"(at[i]), "s"(base), "{m0}"(to + 16 * kThreads * i)
                   : "memory");
  }
};
// Waits until at most n of this wave's copies are under way.
template <int n>
__device__ __forceinline__ void landed() {
  static_assert(n < 64, "counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}

// Eight values of a row, at any address that holds such values (16-byte accesses
// need no alignment here).
template <typename T>
struct Eight {
  static constexpr int kWords = 8 * (int)sizeof(T) / 4;
  uint32_t w[kWords];
};
struct __attribute__((packed, aligned(2))) Packed16 {
  uint32_t w[4];
};
struct __attribute__((packed, aligned(2))) Packed8 {
  uint32_t w[2];
};
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T *p) {
  Eight<T> o;
#pragma unroll
  for (int i = 0; i < Eight<T>::kWords / 4; ++i) {
    const Packed16 v = ((const NSFPS_GLOBAL_SEQ Packed16 *)p)[i];
#pragma unroll
    for (int k = 0; k < 4; ++k) o.w[4 * i + k] = v.w[k];
  }
  return o;
}
// its first n, n below 8, one after another
template <typename T>
__device__ __forceinline__ Eight<T> load_some(const T *p, uint32_t n) {
  Eight<T> o = {};
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k)
    if (k < n) {
      const Raw<T, 1> v = load_raw<T, 1>(p + k);
      if constexpr (sizeof(T) == 4)
        o.w[k] = v.w[0];
      else
        o.w[k / 2] |= v.w[0] << (16 * (k % 2));
    }
  return o;
}
// The values from number n on, zeros behind them; all zeros from 8 on.
template <typename T>
__device__ __forceinline__ void drop(Eight<T> &v, uint32_t n) {
  constexpr int N = Eight<T>::kWords;
  constexpr uint32_t kWordsOf4 = sizeof(T);  // words of four values
#pragma unroll
  for (uint32_t step = 4; step >= (sizeof(T) == 4 ? 1 : 2); step /= 2) {
    const int words = step * kWordsOf4 / 4;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t from = i + words < N ? v.w[i + words] : 0u;
      v.w[i] = n & step ? from : v.w[i];
    }
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t next = i + 1 < N ? v.w[i + 1] : 0u;
      v.w[i] = n & 1 ? v.w[i] >> 16 | next << 16 : v.w[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v.w[i] = n < 8 ? v.w[i] : 0u;
}

// The first n values, zeros behind them.
template <typename T>
__device__ __forceinline__ void keep(Eight<T> &v, uint32_t n) {
#pragma unroll
  for (uint32_t i = 0; i < Eight<T>::kWords; ++i) {
    if constexpr (sizeof(T) == 4)
      v.w[i] = i < n ? v.w[i] : 0u;
    else
      v.w[i] &= (2 * i < n ? 0xffffu : 0u) | (2 * i + 1 < n ? 0xffff0000u : 0u);
  }
}

// What may be read of a tile's rows beside the values inside.
enum class Ends {
  kWide,    // nothing; rows have 8 values or more: a row's last 8 are fetched for its end
  kNarrow,  // nothing; rows have fewer than 8 values, which come one after another
  kPadded,  // as many values as the tile is wide, of whatever they are
};

// A tile through registers: ROWS x COLS of memory, fetched while the tiles before
// it are worked on, split into P planes and put.  What lies outside is zeros: the
// last row, or other values, are fetched in its place and put() mends that.  (A
// load that waits for a condition, or whose value is used where it stands, would
// hold up those behind it: so it is with kNarrow.)
template <typename T, int ROWS, int COLS, int kThreads, Ends kEnds>
struct Stage {
  static constexpr int kPer = ROWS * COLS / 8 / kThreads, kVecs = COLS / 8;
  static_assert(kPer >= 1, "tile too small");
  Eight<T> v[kPer];
  uint32_t tag[kPer];   // of the pieces' rows
  uint32_t rows, cols;  // inside

  // at: the tile's first value; nrows, ncols: how many of it are inside, at least 1.
  // tag_of(row): what put() decides by whether the row is wanted.
  template <typename F>
  __device__ __forceinline__ void fetch(const T *at, uint64_t ld, uint32_t nrows, uint32_t ncols,
                                        F tag_of) {
    rows = nrows;
    cols = min(ncols, (uint32_t)COLS);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + kThreads * i, r = min(e / kVecs, rows - 1), c = e % kVecs * 8;
      const T *row = at + r * ld;
      if constexpr (kEnds == Ends::kWide)
        v[i] = load_eight<T>(row + min((int32_t)c, (int32_t)cols - 8));
      else if constexpr (kEnds == Ends::kNarrow)
        v[i] = load_some<T>(row, c ? 0u : cols);
      else
        v[i] = load_eight<T>(row + c);
      tag[i] = tag_of(r);
    }
    __builtin_amdgcn_sched_barrier(0);  // asked for now, and in order: put() counts on both
  }
  // kT: columns of a Col tile; plane: values of a plane in LDS
  template <int kT, int kTerms, bool kCol, int P, typename F>
  __device__ __forceinline__ void put(bf16 *tile, uint32_t plane, F wanted) {
    const bool whole = rows >= (uint32_t)ROWS && cols >= (uint32_t)COLS;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + kThreads * i, r = e / kVecs, c = e % kVecs * 8;
      if (!whole) {  // the same for all lanes; most tiles are
        if constexpr (kEnds == Ends::kWide)
          drop<T>(v[i], c + 8 > cols ? c + 8 - cols : 0u);
        else if constexpr (kEnds == Ends::kPadded)
          keep<T>(v[i], cols > c ? cols - c : 0u);
        if (r >= rows) v[i] = Eight<T>{};
      }
      if (!wanted(tag[i])) v[i] = Eight<T>{};
      bf16 *const to = tile + piece_at<kT, kTerms, kCol>(r, c);
      if constexpr (sizeof(T) == 2) {
        static_assert(P == 1, "a bfloat16 value is one term");
        *(u32x4 *)to = u32x4{v[i].w[0], v[i].w[1], v[i].w[2], v[i].w[3]};
      } else {
        f32x4 a, b;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          a[k] = __uint_as_float(v[i].w[k]), b[k] = __uint_as_float(v[i].w[4 + k]);
        const Terms<bf16, P> ta = split<bf16, P>(a), tb = split<bf16, P>(b);
#pragma unroll
        for (int p = 0; p < P; ++p)
          *(bf16x8 *)(to + p * plane) =
              __builtin_shufflevector(ta.q[p], tb.q[p], 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
  }
};

// The products of planes that make one product to the bits of the planes, the
// smallest first: plane of m, plane of n.
template <int PM, int PN>
struct Passes;
template <>
struct Passes<1, 1> {
  static constexpr int kN = 1, m[kN] = {0}, n[kN] = {0};
};
template <>
struct Passes<2, 1> {
  static constexpr int kN = 2, m[kN] = {1, 0}, n[kN] = {0, 0};
};
template <>
struct Passes<3, 3> {  // to 24 bits: what is left out is below 2^-24 of the product
  static constexpr int kN = 6, m[kN] = {2, 0, 1, 1, 0, 0}, n[kN] = {0, 2, 1, 0, 1, 0};
};

// WM x WN waves of MT x NT tiles of 16 x 16 sums; stages of kTerms terms, PM and
// PN planes.
template <int WM, int WN, int MT, int NT, int kTerms, int PM, int PN, bool kMCol, bool kNCol,
          bool kPerm>
struct Product {
  static constexpr int kMT = MT, kNT = NT;
  static constexpr int kM = 16 * WM * MT, kN = 16 * WN * NT, kThreads = 64 * WM * WN;
  static_assert(!kPerm || (NT % 2 == 0 && !kNCol), "layout");
  static constexpr int kMPlane = kM * kTerms, kNPlane = kN * kTerms;
  struct alignas(16) Lds {
    bf16 m[PM * kMPlane], n[PN * kNPlane];
  };
  typedef f32x4 Sum[MT][NT];

  static __device__ __forceinline__ uint32_t wave_id() {
    return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  }
  static __device__ __forceinline__ uint32_t first_m() { return wave_id() / WN * (16 * MT); }
  static __device__ __forceinline__ uint32_t first_n() { return wave_id() % WN * (16 * NT); }

  // the first of this lane's four columns of tile t
  static __device__ __forceinline__ uint32_t column(int t) {
    const uint32_t g = (threadIdx.x & 63u) >> 4;
    return first_n() + (kPerm ? 32 * (t / 2) + 8 * g + 4 * (t % 2) : 16 * t + 4 * g);
  }
  static __device__ __forceinline__ bf16x8 read_m(const Lds &lds, int p, int t, uint32_t kb) {
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u, m0 = first_m() + 16 * t;
    const bf16 *tile = lds.m + p * kMPlane;
    return kMCol ? read_col<kM>(tile, m0, kb, g, l) : read_row<kTerms>(tile, m0 + l, kb, g);
  }
  static __device__ __forceinline__ bf16x8 read_n(const bf16 *tile, int t, uint32_t kb) {
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u, n0 = first_n();
    return kNCol   ? read_col<kN>(tile, n0 + 16 * t, kb, g, l)
           : kPerm ? read_row<kTerms>(tile, n0 + 32 * (t / 2) + 8 * (l / 4) + 4 * (t % 2) + l % 4, kb, g)
                   : read_row<kTerms>(tile, n0 + 16 * t + l, kb, g);
  }
  static __device__ __forceinline__ void add_block(Sum &sum, const bf16x8 (&m)[PM][MT],
                                                   const bf16x8 (&n)[PN][NT]) {
    typedef Passes<PM, PN> P;
#pragma unroll
    for (int p = 0; p < P::kN; ++p)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(n[P::n[p]][j], m[P::m[p]][i],
                                                              sum[i][j], 0, 0, 0);
  }
  static __device__ __forceinline__ void read_block(const Lds &lds, uint32_t kb,
                                                    bf16x8 (&m)[PM][MT], bf16x8 (&n)[PN][NT]) {
#pragma unroll
    for (int p = 0; p < PM; ++p)
#pragma unroll
      for (int t = 0; t < MT; ++t) m[p][t] = read_m(lds, p, t, kb);
#pragma unroll
    for (int p = 0; p < PN; ++p)
#pragma unroll
      for (int t = 0; t < NT; ++t) n[p][t] = read_n(lds.n + p * kNPlane, t, kb);
  }
  // Adds a stage that is in LDS.
  static __device__ __forceinline__ void add(Sum &sum, const Lds &lds) {
#pragma unroll
    for (uint32_t kb = 0; kb < kTerms / 32; ++kb) {
      bf16x8 m[PM][MT], n[PN][NT];
      read_block(lds, kb, m, n);
      add_block(sum, m, n);
    }
  }
};

}  // namespace seq
}  // namespace nsfps
