// Softmax cross entropy over a large vocabulary, and its gradient.
//
//   z = scale x E^T,  lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_i,target
//   d_iv = dloss_i scale (exp(z_iv - lse_i) - [v is the target]),
//   dx = d E,  dE = d^T x
//
// The logits are never held: the call finds each tile of z on the matrix cores
// and keeps a running maximum and sum of exponentials of every token; the
// gradient finds z again, a piece of the vocabulary at a time, and leaves the
// piece's d in the workspace as an operand of the two products that read it.
//
// Operands of the products are bfloat16 terms.  A float32 value enters as three
// terms whose sum it is, and a product of float32 values as the six products of
// terms that reach 24 bits.  d is rounded to one term (8 bits) where the
// products' results are bfloat16, to two for a float32 table gradient of
// bfloat16 inputs, to three in float32 calls.  Sums are float32 everywhere.
// (Two terms for bfloat16 results too, through registers: the error against 64 bits
// goes from 0.0019 to 0.0017 of the norm at 77 tokens x 313 rows, where probabilities
// are not small, from 0.00165 to 0.00164 at 30 x 19,106; the time from 24.5 to 24.5
// and from 67 to 76 us, at 46 x 241,327 x 79 from 130 to 163.  One is what a result of
// 8 bits is worth.)
//
// The matrix cores bound large calls: the statistics of 16,384 tokens, 262,144
// rows of 256 bfloat16 take 1.96 ms, 1.12 PFLOP/s, as fast as a plain product of
// 8,192^3 (1.13).  Their gradient takes 64 pieces of 4,096 rows: d 62 to 64 us by card
// (its product alone would take 30 at that rate, the 134 MB that it writes 26 at a
// copy's), the two products that read it 70 to 76 us (0.98 to 0.92 PFLOP/s), the sums'
// rows 5.5 us.  64 million values of d a piece: 32, 128 and 256 million were no faster,
// and more than 128 million would not stay in the memory-side cache.  A float32
// call's six products a product: 16,384 tokens, 8,192 rows, width 383 in 2.3 to 2.4
// ms by card, where float32 matrix instructions would need 2.7.  A table's one reading
// bounds calls of few tokens: 7 tokens, 262,144 rows of 256 bfloat16 27 us, 5.0 TB/s.
#include "nsfps_launch.h"
#include "nsfps_product.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

constexpr uint32_t kTile = 128;  // tokens and vocabulary rows of a tile

// rows x cols values, rows ld elements apart
struct Matrix {
  const void *p;
  uint64_t ld;
  uint32_t rows, cols;
};

// The tokens' weights, dloss * scale.  d is held relative to one of them, which the
// products' results get back: where all weights are alike, as for a mean, a
// token's own term is then -(1 - p), which 8 bits hold to 2^-9 and mostly better,
// and not a value whose rounding, the same for every token, would show in all
// results (error against 64 bits up to 0.0032, where the results' own rounding
// leaves 0.0017).
struct Weights {
  const float *dloss;
  const int32_t *targets;
  uint32_t tokens, vocabulary;
  float scale;

  // (loads that wait for no other: all of them are asked for at once)
  __device__ __forceinline__ uint32_t in(uint32_t token) const { return min(token, tokens - 1); }
  __device__ __forceinline__ bool counts(uint32_t token) const {
    const uint32_t target = (uint32_t)targets[in(token)];
    return token < tokens && target < vocabulary;
  }
  // That of the first of 64 tokens that counts, if it is of an ordinary size.
  __device__ __forceinline__ float reference() const {
    const uint32_t lane = threadIdx.x & 63u;
    const float own = dloss[in(lane)] * scale, w = counts(lane) ? own : 0.f;
    const uint64_t fit = __ballot(fabsf(w) >= 0x1p-30f && fabsf(w) <= 0x1p30f);
    return fit ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), __builtin_ctzll(fit)))
               : 1.f;
  }
};

// ---- tiles of z

// Tiles of tokens and of a piece's vocabulary; how many of the latter a workgroup
// takes one after another, and such sweeps.
struct Tiling {
  uint32_t ttiles, vtiles, sweep, sweeps;
};

struct LogitDev {
  Matrix x, e;                // e: the piece (x may be padded)
  Tiling tiles;
  float scale2;               // scale * log2(e)
  double to_2;                // exponents of an lse: scale2 / scale
  // statistics
  float2 *parts;              // [sweeps][part_stride]: maximum and sum, in powers of two
  uint64_t part_stride;
  // gradient
  const float *lse;
  Weights weights;
  uint32_t row0;              // the piece's first
  void *d;                    // [tokens][d_ld] (kDirect: whole tiles of tokens)
  uint64_t d_ld;
};

// Workgroup w's tile of tokens and sweep, the latter as vocabulary tiles of N rows:
// tokens change fastest, within groups that share sweeps, so that workgroups of one
// XCD read the same rows.
template <uint32_t N, uint32_t kUnit>
__device__ __forceinline__ bool logit_item(const LogitDev &a, uint32_t &ttile, uint32_t &sweep,
                                           uint32_t &first, uint32_t &last) {
  const uint32_t work = a.tiles.ttiles * a.tiles.sweeps, per = (work + 7) / 8;
  const uint32_t w = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || w >= work) return false;
  constexpr uint32_t kGroup = 8;
  const uint32_t whole = kGroup * a.tiles.sweeps, group = w / whole, t0 = group * kGroup;
  const uint32_t size = min(kGroup, a.tiles.ttiles - t0), in = w - group * whole;
  ttile = t0 + in % size;
  sweep = in / size;
  first = kUnit / N * (sweep * a.tiles.sweep);
  last = kUnit / N * min(sweep * a.tiles.sweep + a.tiles.sweep, a.tiles.vtiles);
  return true;
}

// The tiles of z that a workgroup walks, one after another; epilogue.whole(sum,
// tile) has each.  Operands through registers: any rows, either type.
// kTiles: 16 x 16 tiles of a wave either way.
template <typename T, int P, bool kPerm, Ends kEnds, int kTiles>
struct StagedLogits {  // (every row is wanted)
  static constexpr int kTerms = P == 1 ? 64 : 32;
  static constexpr int kAhead = 2;  // stages under way
  typedef Product<2, 2, kTiles, kTiles, kTerms, P, P, false, false, kPerm> Prod;
  static constexpr uint32_t kUnit = Prod::kN;
  typedef typename Prod::Lds Lds;
  static constexpr bool kDirect = false;

  template <typename F>
  static __device__ __forceinline__ void walk(const LogitDev &a, Lds &lds, uint32_t ttile,
                                              uint32_t first, uint32_t last, F &epilogue) {
    Stage<T, Prod::kM, kTerms, 256, kEnds> sx[kAhead], se[kAhead];
    const uint32_t width = a.x.cols, steps = ceil_div(width, kTerms);
    const uint32_t t0 = ttile * Prod::kM;
    const T *const x = (const T *)a.x.p + (uint64_t)t0 * a.x.ld;
    const auto none = [](uint32_t) { return 0u; };
    const auto all = [](uint32_t) { return true; };
    uint32_t tile = first, k = 0;  // of the stage fetched next
    const auto fetch = [&](int to) {  // past the end the last tile again
      const uint32_t v0 = min(min(tile, last - 1) * Prod::kN, a.e.rows - 1);
      sx[to].fetch(x + k * kTerms, a.x.ld, a.x.rows - t0, width - k * kTerms, none);
      se[to].fetch((const T *)a.e.p + (uint64_t)v0 * a.e.ld + k * kTerms, a.e.ld, a.e.rows - v0,
                   width - k * kTerms, none);
      if (++k == steps) k = 0, ++tile;
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(i);
    wait_loads();
    typename Prod::Sum sum = {};
    uint32_t s = 0;
    for (uint32_t t = first; t < last;) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (t >= last) break;
        __syncthreads();
        sx[i].template put<Prod::kM, kTerms, false, P>(lds.m, Prod::kMPlane, all);
        se[i].template put<Prod::kN, kTerms, false, P>(lds.n, Prod::kNPlane, all);
        __syncthreads();
        fetch(i);
        Prod::add(sum, lds);
        if (++s == steps) {
          epilogue.whole(sum, t);
#pragma unroll
          for (int q = 0; q < Prod::kMT; ++q)
#pragma unroll
            for (int j = 0; j < Prod::kNT; ++j) sum[q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
          s = 0;
          ++t;
        }
      }
    }
  }
};

// The same straight to LDS: bfloat16, rows of whole 64s at 16-byte boundaries.
// Rows past the end are the last one again.
struct DirectLogits {
  typedef Product<2, 2, 4, 4, 64, 1, 1, false, false, true> Prod;
  struct Lds {
    typename Prod::Lds buf[2];
  };
  static constexpr bool kDirect = true;
  static constexpr uint32_t kUnit = kTile;

  template <typename F>
  static __device__ __forceinline__ void walk(const LogitDev &a, Lds &lds, uint32_t ttile,
                                              uint32_t first, uint32_t last, F &epilogue) {
    Feed<kTile, 64, false, 256> fx, fe;
    const uint32_t steps = a.x.cols / 64;
    const bf16 *const x = (const bf16 *)a.x.p + (uint64_t)ttile * kTile * a.x.ld;
    fx.start(a.x.ld, a.x.rows - ttile * kTile);
    fe.start(a.e.ld, ~0u);
    uint32_t tile = first, k = 0, buf = 0;  // of the stage issued next
    const auto issue = [&](uint32_t b) {
      const uint32_t v0 = min(tile * kTile, a.e.rows - 1);
      if (k == 0 && v0 + kTile > a.e.rows) fe.start(a.e.ld, a.e.rows - v0);
      fx.issue(lds.buf[b].m, x + 64 * k);
      fe.issue(lds.buf[b].n, (const bf16 *)a.e.p + (uint64_t)v0 * a.e.ld + 64 * k);
      if (++k == steps) k = 0, ++tile;
    };
    issue(0);
    wait_loads();
    for (uint32_t t = first; t < last; ++t) {
      typename Prod::Sum sum = {};
      for (uint32_t s = 0; s < steps; ++s) {
        landed<0>();
        __syncthreads();
        if (tile < last) issue(buf ^ 1);
        Prod::add(sum, lds.buf[buf]);
        buf ^= 1;
      }
      epilogue.whole(sum, t);
    }
  }
};

// The same for widths of up to 256 and long sweeps: a workgroup's tokens stay in
// registers, so that LDS, which gives 128 bytes a cycle, is read for the vocabulary
// alone (with both from LDS those reads and the copies took half as long again as
// the products).  Three stages are under way while a fourth is worked on.
template <int kTerms, int kSteps>
struct ResidentLogits {
  typedef Product<2, 2, 4, 2, kTerms, 1, 1, false, false, true> Prod;
  struct alignas(16) Lds {
    bf16 buf[4][Prod::kN * kTerms];
  };
  static constexpr bool kDirect = true;
  static constexpr uint32_t kUnit = kTile;

  template <typename F>
  static __device__ __forceinline__ void walk(const LogitDev &a, Lds &lds, uint32_t ttile,
                                              uint32_t first, uint32_t last, F &epilogue) {
    constexpr int kBlocks = kTerms / 32;
    Feed<Prod::kN, kTerms, false, 256> fe;
    constexpr int kCopies = fe.kPer;
    fe.start(a.e.ld, ~0u);
    uint32_t tile = first, k = 0, to = 0, buf = 0;
    const auto issue = [&] {  // past the end the last tile again: counts stay the same
      const uint32_t v0 = min(min(tile, last - 1) * Prod::kN, a.e.rows - 1);
      if (v0 + Prod::kN > a.e.rows) fe.start(a.e.ld, a.e.rows - v0);
      fe.issue(lds.buf[to], (const bf16 *)a.e.p + (uint64_t)v0 * a.e.ld + kTerms * k);
      if (++k == kSteps) k = 0, ++tile;
      to = (to + 1) % 4;
    };
    issue();
    issue();
    issue();
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
    bf16x8 x[kSteps][kBlocks][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = min(ttile * kTile + Prod::first_m() + 16 * i + l, a.x.rows - 1);
      const bf16 *row = (const bf16 *)a.x.p + r * a.x.ld + 8 * g;
#pragma unroll
      for (int k = 0; k < kBlocks * kSteps; ++k)
        x[k / kBlocks][k % kBlocks][i] = *(const NSFPS_GLOBAL_SEQ bf16x8 *)(row + 32 * k);
    }
    wait_loads();
    for (uint32_t t = first; t < last; ++t) {
      typename Prod::Sum sum = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        landed<2 * kCopies>();
        __syncthreads();
        issue();
#pragma unroll
        for (uint32_t kb = 0; kb < kBlocks; ++kb) {
          const bf16x8 n[1][2] = {
              {Prod::read_n(lds.buf[buf], 0, kb), Prod::read_n(lds.buf[buf], 1, kb)}};
          const bf16x8 m[1][4] = {{x[s][kb][0], x[s][kb][1], x[s][kb][2], x[s][kb][3]}};
          Prod::add_block(sum, m, n);
        }
        buf = (buf + 1) % 4;
      }
      epilogue.whole(sum, t);
    }
    landed<0>();
  }
};

__device__ __forceinline__ void join_stats(float &m, float &s, float m2, float s2) {
  const float top = fmaxf(m, m2), at = top == -INFINITY ? 0.f : top;
  s = s * exp2_fast(m - at) + s2 * exp2_fast(m2 - at);
  m = top;
}

// The factor that makes a power of two's exponent of a logit without its scale, and
// without its sign.  (Not 0: -infinity times 0 would be NaN.)
__host__ __device__ __forceinline__ float exponent_by(float scale2) {
  return fmaxf(fabsf(scale2), 1e-38f);
}

// Running maximum and sum of a lane's columns, for its tokens.
template <typename Prod>
struct Stats {
  const LogitDev &a;
  const float by;
  float top[Prod::kMT], sum[Prod::kMT];

  __device__ __forceinline__ explicit Stats(const LogitDev &args)
      : a(args), by(exponent_by(args.scale2)) {
#pragma unroll
    for (int i = 0; i < Prod::kMT; ++i) top[i] = -INFINITY, sum[i] = 0.f;
  }
  // nothing to do but part(): no column past the end, no sign to turn
  __device__ __forceinline__ bool plain(uint32_t tile) const {
    return (tile + 1) * Prod::kN <= a.e.rows && a.scale2 >= 0.f;
  }
  __device__ __forceinline__ void part(const typename Prod::Sum &z, int i) {
    float m = z[i][0][0];
#pragma unroll
    for (int j = 0; j < Prod::kNT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, z[i][j][r]);
    m = fmaxf(top[i], m * by);
    const float at = m == -INFINITY ? 0.f : m;
    float s = sum[i] * exp2_fast(top[i] - at);
#pragma unroll
    for (int j = 0; j < Prod::kNT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) s += exp2_fast(fmaf(z[i][j][r], by, -at));
    top[i] = m;
    sum[i] = s;
  }
  __device__ __forceinline__ void whole(typename Prod::Sum &z, uint32_t tile) {
    if (!plain(tile)) {
#pragma unroll
      for (int i = 0; i < Prod::kMT; ++i)
#pragma unroll
        for (int j = 0; j < Prod::kNT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (a.scale2 < 0.f) z[i][j][r] = -z[i][j][r];
            if (tile * Prod::kN + Prod::column(j) + r >= a.e.rows) z[i][j][r] = -INFINITY;
          }
    }
#pragma unroll
    for (int i = 0; i < Prod::kMT; ++i) part(z, i);
  }
};

template <typename Logits>
__global__ __launch_bounds__(256, 2) void k_loss_stats(LogitDev a) {
  typedef typename Logits::Prod Prod;
  __shared__ typename Logits::Lds lds;
  __shared__ float2 s_part[2][Prod::kM];
  uint32_t ttile, sweep, first, last;
  if (!logit_item<Prod::kN, Logits::kUnit>(a, ttile, sweep, first, last)) return;
  const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % 2;
  Stats<Prod> o(a);
  Logits::walk(a, lds, ttile, first, last, o);
#pragma unroll
  for (int i = 0; i < Prod::kMT; ++i) {
#pragma unroll
    for (int off = 16; off < 64; off <<= 1)
      join_stats(o.top[i], o.sum[i], __shfl_xor(o.top[i], off, 64), __shfl_xor(o.sum[i], off, 64));
    if (g == 0) s_part[wn][Prod::first_m() + 16 * i + l] = make_float2(o.top[i], o.sum[i]);
  }
  __syncthreads();
  const uint32_t token = ttile * Prod::kM + threadIdx.x;
  if (threadIdx.x < Prod::kM && token < a.x.rows) {
    float2 v = s_part[0][threadIdx.x];
    join_stats(v.x, v.y, s_part[1][threadIdx.x].x, s_part[1][threadIdx.x].y);
    a.parts[sweep * a.part_stride + token] = v;
  }
}

template <typename T>
__device__ __forceinline__ float value(const Eight<T> &v, int k) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(v.w[k]);
  return __uint_as_float(k % 2 ? v.w[k / 2] & 0xffff0000u : v.w[k / 2] << 16);
}

// lse and loss: a workgroup has `group` tokens (a power of two, at most 16), 256 /
// group runs of parts for each; then as many lanes, a wave at most, find the logit of
// a token's target.  Its bytes bound it in large calls (14,990 tokens x 147 rows x
// width 954 float32: 14 us), else its three loads one after another (4 us).
template <typename T>
__global__ __launch_bounds__(256) void k_loss_join(const float2 *__restrict__ parts, uint32_t nparts,
                                                   uint64_t part_stride, uint32_t group, Matrix x,
                                                   Matrix table, float scale, double to_e,
                                                   const int32_t *__restrict__ targets,
                                                   float *__restrict__ loss,
                                                   float *__restrict__ lse) {
  __shared__ float2 s_part[4][16];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, tokens = x.rows;
  for (uint32_t t0 = blockIdx.x * group; t0 < tokens; t0 += gridDim.x * group) {
    const uint32_t mine = min(t0 + lane % group, tokens - 1), runs = 256 / group;
    float m = -INFINITY, s = 0.f;
    for (uint32_t p = threadIdx.x / group; p < nparts; p += runs) {
      const float2 v = parts[p * part_stride + mine];
      join_stats(m, s, v.x, v.y);
    }
    for (uint32_t off = group; off < 64; off <<= 1)
      join_stats(m, s, __shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
    if (lane < group) s_part[wave][lane] = make_float2(m, s);
    __syncthreads();
    const uint32_t per = min(256 / group, 64u), i = threadIdx.x / per, token = t0 + i;
    if (i < group && token < tokens) {
      const uint32_t target = (uint32_t)targets[token], own = threadIdx.x % per;
      float dot = 0.f;
      if (target < table.rows) {
        const T *xr = (const T *)x.p + token * x.ld, *er = (const T *)table.p + target * table.ld;
        const uint32_t whole = x.cols / 8, c = 8 * whole + own;
#pragma unroll 2
        for (uint32_t q = own; q < whole; q += per) {
          const Eight<T> u = load_eight<T>(xr + 8 * q), v = load_eight<T>(er + 8 * q);
#pragma unroll
          for (int k = 0; k < 8; ++k) dot = fmaf(value(u, k), value(v, k), dot);
        }
        if (c < x.cols) {
          float u[1], v[1];
          load_f32<T, 1>(xr + c, u);
          load_f32<T, 1>(er + c, v);
          dot = fmaf(u[0], v[0], dot);
        }
      }
      for (uint32_t off = 1; off < per; off <<= 1) dot += __shfl_xor(dot, off, 64);
      float2 v = s_part[0][i];
#pragma unroll
      for (int k = 1; k < 4; ++k) join_stats(v.x, v.y, s_part[k][i].x, s_part[k][i].y);
      // In float64, for the logits may be far above the loss.  The largest exponent gets
      // back its logit by to_e, the inverse of by (Stats) with by's rounding; the sum's
      // exponents keep that rounding, 2^-24 of how far the logits lie below the largest.
      int power;
      const float part = frexpf(v.y, &power);
      const double all = (v.x == -INFINITY ? -INFINITY : v.x * to_e) +
                         (power + (double)log2f(part)) * 0.693147180559945309417;
      if (own == 0) {
        lse[token] = (float)all;
        loss[token] = target < table.rows ? (float)(all - (double)scale * dot) : 0.f;
      }
    }
    __syncthreads();
  }
}

// A piece's d, as D, for a lane's tokens.
template <typename Logits, typename D>
struct Derivatives {
  typedef typename Logits::Prod Prod;
  const LogitDev &a;
  const uint32_t token0;
  float lse2[Prod::kMT], weight[Prod::kMT];
  uint32_t target[Prod::kMT];  // in the piece
  bool counts[Prod::kMT];

  __device__ __forceinline__ Derivatives(const LogitDev &args, uint32_t ttile)
      : a(args), token0(ttile * Prod::kM + Prod::first_m() + (threadIdx.x & 15u)) {
    const float reference = a.weights.reference();
#pragma unroll
    for (int i = 0; i < Prod::kMT; ++i) {
      const uint32_t token = token0 + 16 * i, at = a.weights.in(token);
      const float lse = (float)(a.lse[at] * a.to_2),
                  own = a.weights.dloss[at] * a.weights.scale / reference;
      counts[i] = a.weights.counts(token);
      lse2[i] = counts[i] ? lse : 0.f;
      weight[i] = counts[i] ? own : 0.f;
      target[i] = counts[i] ? (uint32_t)a.weights.targets[at] - a.row0 : ~0u;
    }
  }
  // no column past the end, no token's target, and no token that does not count
  // (whose row is zeros where tiles go straight to LDS, and so is its d)
  __device__ __forceinline__ bool plain(uint32_t tile) const {
    bool special = false;
#pragma unroll
    for (int i = 0; i < Prod::kMT; ++i)
      special |= target[i] - tile * Prod::kN < Prod::kN || (!Logits::kDirect && !counts[i]);
    return (tile + 1) * Prod::kN <= a.e.rows && !__any(special);
  }
  __device__ __forceinline__ void values(const typename Prod::Sum &z, int i,
                                         float (&d)[4 * Prod::kNT]) const {
#pragma unroll
    for (int j = 0; j < Prod::kNT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        d[4 * j + r] = exp2_fast(fmaf(z[i][j][r], a.scale2, -lse2[i])) * weight[i];
  }
  // 16 bytes a lane, the four lanes of a row beside each other
  __device__ __forceinline__ void store(uint32_t tile, int i, const float (&d)[4 * Prod::kNT]) const {
    if (!Logits::kDirect && token0 + 16 * i >= a.x.rows) return;
    D *const out = (D *)a.d + (uint64_t)(token0 + 16 * i) * a.d_ld + tile * Prod::kN;
    constexpr int V = kWide<D>;
#pragma unroll
    for (int k = 0; k < 4 * Prod::kNT; k += V) {
      float o[V];
#pragma unroll
      for (int q = 0; q < V; ++q) o[q] = d[k + q];
      store_f32<D, V>(out + Prod::column(k / 4), o);
    }
  }
  __device__ __forceinline__ void whole(const typename Prod::Sum &z, uint32_t tile) const {
    const bool simple = plain(tile);
#pragma unroll
    for (int i = 0; i < Prod::kMT; ++i) {
      float d[4 * Prod::kNT];
      values(z, i, d);
      if (!simple) {
#pragma unroll
        for (int j = 0; j < Prod::kNT; ++j) {
          const uint32_t v = tile * Prod::kN + Prod::column(j);
#pragma unroll
          for (uint32_t r = 0; r < 4; ++r) {
            if (target[i] == v + r)
              d[4 * j + r] =
                  (exp2_fast(fmaf(z[i][j][r], a.scale2, -lse2[i])) - 1.f) * weight[i];
            if (!counts[i] || v + r >= a.e.rows) d[4 * j + r] = 0.f;
          }
        }
      }
      store(tile, i, d);
    }
  }
};

template <typename Logits, typename D>
__global__ __launch_bounds__(256, 2) void k_loss_d(LogitDev a) {
  __shared__ typename Logits::Lds lds;
  uint32_t ttile, sweep, first, last;
  if (!logit_item<Logits::Prod::kN, Logits::kUnit>(a, ttile, sweep, first, last)) return;
  Derivatives<Logits, D> o(a, ttile);
  Logits::walk(a, lds, ttile, first, last, o);
}

// ---- the products of d

struct ProductDev {
  Matrix m, n;           // as they lie in memory
  uint32_t mtiles, ntiles;
  uint32_t terms;        // k from 0 on
  uint32_t per, splits;  // k of a split (whole 64s), splits
  // the result: either rows of it, or the splits' sums
  void *out;
  uint64_t out_ld;
  uint32_t out_rows, out_cols, out_dtype;
  float *sums;           // [splits][rows][sums_ld], null: out is written
  uint64_t sums_split, sums_ld;
  uint32_t add;          // to what sums holds
  uint32_t out_lanes;    // for a value of the result, a power of two of at most 64
  Weights weights;
};

// at any address of such values
__device__ __forceinline__ void store_four(float *p, const float (&v)[4]) {
  *(NSFPS_GLOBAL_SEQ Packed16 *)p = Packed16{{__float_as_uint(v[0]), __float_as_uint(v[1]),
                                              __float_as_uint(v[2]), __float_as_uint(v[3])}};
}
__device__ __forceinline__ void store_four(bf16 *p, const float (&v)[4]) {
  *(NSFPS_GLOBAL_SEQ Packed8 *)p =
      Packed8{{(uint32_t)bf16_bits(v[0]) | (uint32_t)bf16_bits(v[1]) << 16,
               (uint32_t)bf16_bits(v[2]) | (uint32_t)bf16_bits(v[3]) << 16}};
}

template <typename Prod>
__device__ __forceinline__ void put_result(const ProductDev &a, const typename Prod::Sum &sum,
                                           uint32_t m0, uint32_t n0, uint32_t split) {
  constexpr int MT = Prod::kMT, NT = Prod::kNT;
  const float by = a.sums ? 1.f : a.weights.reference();
  const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
  const uint32_t m = m0 + Prod::first_m() + l, n = n0 + Prod::first_n() + 4 * g;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t row = m + 16 * i, col = n + 16 * j;
      if (row >= a.out_rows || col >= a.out_cols) continue;
      if (a.sums) {
        NSFPS_GLOBAL_SEQ f32x4 *at =
            (NSFPS_GLOBAL_SEQ f32x4 *)(a.sums + split * a.sums_split + row * a.sums_ld + col);
        *at = a.add ? *at + sum[i][j] : sum[i][j];
        continue;
      }
      const float v[4] = {sum[i][j][0] * by, sum[i][j][1] * by, sum[i][j][2] * by, sum[i][j][3] * by};
      const auto store = [&](auto t) {
        using T = decltype(t);
        T *const out = (T *)a.out + row * a.out_ld + col;
        if (col + 4 <= a.out_cols) {
          store_four(out, v);
        } else {
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {
            const float one[1] = {v[k]};
            if (col + k < a.out_cols) store_f32<T, 1>(out + k, one);
          }
        }
      };
      if (a.out_dtype == NSFPS_F32)
        store(float());
      else
        store(bf16());
    }
}

struct ProductItem {
  uint32_t mt, nt, split, k0, k1;  // from k0 to k1, nothing where k0 is not below k1
};
__device__ __forceinline__ ProductItem product_item(const ProductDev &a, uint32_t w) {
  ProductItem o;
  o.nt = w % a.ntiles;
  o.mt = w / a.ntiles % a.mtiles;
  o.split = w / a.ntiles / a.mtiles;
  o.k0 = min(o.split * a.per, a.terms);
  o.k1 = min(o.k0 + a.per, a.terms);
  return o;
}

// M's terms along its rows (dx) or down its columns (dE), N's down its columns.
template <typename TM, int PM, typename TN, int PN, int NT, bool kMCol, Ends kEnds>
struct StagedProduct {
  static constexpr int kTerms = PM * PN == 1 ? 64 : 32, kAhead = 2;
  typedef Product<2, 2, 4, NT, kTerms, PM, PN, kMCol, true, false> Prod;
  static constexpr int kMRows = kMCol ? kTerms : Prod::kM, kMCols = kMCol ? Prod::kM : kTerms;

  static __device__ __forceinline__ void run(const ProductDev &a, typename Prod::Lds &lds,
                                             uint32_t w) {
    const ProductItem it = product_item(a, w);
    const uint32_t m0 = it.mt * Prod::kM, n0 = it.nt * Prod::kN;
    Stage<TM, kMRows, kMCols, 256, Ends::kPadded> sm[kAhead];
    Stage<TN, kTerms, Prod::kN, 256, kEnds> sn[kAhead];
    uint32_t k = it.k0;
    const auto fetch = [&](int to) {  // past the end the last stage again
      const uint32_t at = min(k, (it.k1 - 1) / kTerms * kTerms);
      const uint32_t mr = kMCol ? at : m0, mc = kMCol ? m0 : at;
      sm[to].fetch((const TM *)a.m.p + (uint64_t)mr * a.m.ld + mc, a.m.ld,
                   (kMCol ? a.terms : a.m.rows) - mr, (kMCol ? a.m.cols : a.terms) - mc,
                   [](uint32_t) { return 0u; });
      sn[to].fetch((const TN *)a.n.p + (uint64_t)at * a.n.ld + n0, a.n.ld, a.terms - at,
                   a.n.cols - n0, [&](uint32_t r) {
                     return kMCol ? (uint32_t)a.weights.targets[min(at + r, a.terms - 1)] : 0u;
                   });
      k += kTerms;
    };
    typename Prod::Sum sum = {};
    if (it.k0 < it.k1) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fetch(i);
      for (uint32_t s = it.k0; s < it.k1;) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (s >= it.k1) break;
          __syncthreads();
          sm[i].template put<Prod::kM, kTerms, kMCol, PM>(lds.m, Prod::kMPlane,
                                                          [](uint32_t) { return true; });
          sn[i].template put<Prod::kN, kTerms, true, PN>(
              lds.n, Prod::kNPlane,
              [&](uint32_t target) { return !kMCol || target < a.weights.vocabulary; });
          __syncthreads();
          fetch(i);
          Prod::add(sum, lds);
          s += kTerms;
        }
      }
    }
    put_result<Prod>(a, sum, m0, n0, it.split);
  }
};

// Straight to LDS: bfloat16, M and N whole tiles (rows of N past its end are its
// last again, and meet zeros of M).  Of three places in LDS one is read and two are
// under way, for d comes from beyond the L2 caches.
template <int WM, int WN, int MT, bool kMCol>
struct DirectProduct {
  static constexpr uint32_t kTerms = 64, kPlaces = 3;
  typedef Product<WM, WN, MT, 4, kTerms, 1, 1, kMCol, true, false> Prod;
  struct Lds {
    typename Prod::Lds buf[kPlaces];
  };

  static __device__ __forceinline__ void run(const ProductDev &a, Lds &lds, uint32_t w) {
    const ProductItem it = product_item(a, w);
    const uint32_t m0 = it.mt * Prod::kM, n0 = it.nt * Prod::kN;
    Feed<Prod::kM, kTerms, kMCol, Prod::kThreads> fm;
    Feed<Prod::kN, kTerms, true, Prod::kThreads> fn;
    constexpr int kCopies = fm.kPer + fn.kPer;
    const bf16 *const m = (const bf16 *)a.m.p + (kMCol ? m0 : (uint64_t)m0 * a.m.ld);
    const bf16 *const n = (const bf16 *)a.n.p + n0;
    fm.start(a.m.ld, ~0u);
    fn.start(a.n.ld, ~0u);
    uint32_t k = it.k0, to = 0, buf = 0;
    const auto issue = [&] {  // past the end the last stage again: counts stay the same
      const uint32_t at = min(k, (it.k1 - 1) & ~(kTerms - 1));
      if (at + kTerms > a.n.rows) fn.start(a.n.ld, a.n.rows - at);
      fm.issue(lds.buf[to].m, m + (kMCol ? (uint64_t)at * a.m.ld : at));
      fn.issue(lds.buf[to].n, n + (uint64_t)at * a.n.ld);
      k += kTerms;
      to = to + 1 < kPlaces ? to + 1 : 0;
    };
    typename Prod::Sum sum = {};
    if (it.k0 < it.k1) {
      issue();
      issue();
      for (uint32_t s = it.k0; s < it.k1; s += kTerms) {
        landed<kCopies>();
        __syncthreads();  // the stage before is done with: its place takes the next
        issue();
        Prod::add(sum, lds.buf[buf]);
        buf = buf + 1 < kPlaces ? buf + 1 : 0;
      }
      landed<0>();
    }
    put_result<Prod>(a, sum, m0, n0, it.split);
  }
};

// dx and dE of a piece in one launch, one workgroup an item of either.
__device__ __forceinline__ bool product_work(const ProductDev &dx, const ProductDev &de,
                                             uint32_t &w, bool &is_dx) {
  const uint32_t first = dx.mtiles * dx.ntiles * dx.splits,
                 work = first + de.mtiles * de.ntiles * de.splits, per = (work + 7) / 8;
  w = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || w >= work) return false;
  is_dx = w < first;
  if (!is_dx) w -= first;
  return true;
}

template <typename TD, int PDX, int PDE, typename T, int P, int NT, Ends kEnds>
__global__ __launch_bounds__(256, 2) void k_loss_products(ProductDev dx, ProductDev de) {
  typedef StagedProduct<TD, PDX, T, P, NT, false, kEnds> X;
  typedef StagedProduct<TD, PDE, T, P, NT, true, kEnds> E;
  __shared__ union {
    typename X::Prod::Lds x;
    typename E::Prod::Lds e;
  } lds;
  uint32_t w;
  bool is_dx;
  if (!product_work(dx, de, w, is_dx)) return;
  if (is_dx)
    X::run(dx, lds.x, w);
  else
    E::run(de, lds.e, w);
}

template <int WM, int WN, int MT>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_loss_products_direct(ProductDev dx, ProductDev de) {
  typedef DirectProduct<WM, WN, MT, false> X;
  typedef DirectProduct<WM, WN, MT, true> E;
  extern __shared__ __attribute__((aligned(16))) char s_raw[];
  uint32_t w;
  bool is_dx;
  if (!product_work(dx, de, w, is_dx)) return;
  if (is_dx)
    X::run(dx, *(typename X::Lds *)s_raw, w);
  else
    E::run(de, *(typename E::Lds *)s_raw, w);
}

// Rows for the copies straight to LDS: out_rows x out_cols, zeros past the ends and
// (targets not null) where a row counts for nothing, which may hold anything.
// Memory bound: 16,384 rows of 256 5.8 us.
struct PackDev {
  Matrix in;
  const int32_t *targets;
  uint32_t vocabulary, out_cols;
  bf16 *out;
  uint64_t out_rows;
};
// first's rows, second's with blockIdx.y = 1
__global__ __launch_bounds__(256) void k_loss_pack(PackDev first, PackDev second) {
  const PackDev &a = blockIdx.y ? second : first;
  const uint32_t vecs = a.out_cols / 8;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < a.out_rows * vecs;
       i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = i / vecs;
    const uint32_t c = (uint32_t)(i % vecs) * 8;
    Eight<bf16> v = {};
    if (r < a.in.rows && c < a.in.cols &&
        (!a.targets || (uint32_t)a.targets[r] < a.vocabulary)) {
      const bf16 *const row = (const bf16 *)a.in.p + r * a.in.ld + c;
      v = c + 8 <= a.in.cols ? load_eight<bf16>(row) : load_some<bf16>(row, a.in.cols - c);
    }
    *(NSFPS_GLOBAL_SEQ u32x4 *)(a.out + r * a.out_cols + c) = u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
  }
}

// The splits' sums as rows of the result: four values a group of lanes, each of which
// adds every lanes-th split in order, eight loaded together, and then pairs of lanes.
template <typename T>
__device__ __forceinline__ void write_result(const ProductDev &a) {
  const uint32_t vecs = (a.out_cols + 3) / 4;
  const float by = a.weights.reference();
  const uint32_t lanes = a.out_lanes, lane = threadIdx.x % lanes;
  for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
       i < (uint64_t)a.out_rows * vecs; i += (uint64_t)gridDim.x * 256 / lanes) {
    const uint64_t r = i / vecs, c = i % vecs * 4;
    const NSFPS_GLOBAL_SEQ float *from = (const NSFPS_GLOBAL_SEQ float *)(a.sums + r * a.sums_ld + c);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t s0 = lane; s0 < a.splits; s0 += 8 * lanes) {
      f32x4 v[8];
#pragma unroll
      for (uint32_t s = 0; s < 8; ++s)
        v[s] = *(const NSFPS_GLOBAL_SEQ f32x4 *)(from +
                                                 min(s0 + s * lanes, a.splits - 1) * a.sums_split);
#pragma unroll
      for (uint32_t s = 0; s < 8; ++s)
        if (s0 + s * lanes < a.splits) sum += v[s];
    }
    for (uint32_t off = 1; off < lanes; off <<= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] += __shfl_xor(sum[k], off, 64);
    if (lane) continue;
    const float o[4] = {sum[0] * by, sum[1] * by, sum[2] * by, sum[3] * by};
    T *const out = (T *)a.out + r * a.out_ld + c;
    if (c + 4 <= a.out_cols) {
      store_four(out, o);
    } else {
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        const float one[1] = {o[k]};
        if (c + k < a.out_cols) store_f32<T, 1>(out + k, one);
      }
    }
  }
}

// first's result, second's with blockIdx.y = 1
__global__ __launch_bounds__(256) void k_loss_out(ProductDev first, ProductDev second) {
  const ProductDev &a = blockIdx.y ? second : first;
  if (a.out_dtype == NSFPS_F32)
    write_result<float>(a);
  else
    write_result<bf16>(a);
}

template <typename T>
__global__ __launch_bounds__(256) void k_loss_zeros(T *__restrict__ out, uint64_t stride,
                                                    uint64_t rows, uint32_t width) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < rows * width;
       i += (uint64_t)gridDim.x * 256)
    out[i / width * stride + i % width] = from_f32<T>(0.f);
}

// ---- the plan of a call

uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }
uint64_t bytes256(uint64_t n) { return up(n, 256); }
uint32_t grid_of(uint64_t threads) {
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(1u << 16, host_ceil_div(threads, 256)));
}
uint32_t xcd_grid(uint64_t work) { return (uint32_t)((work + 7) / 8 * 8); }

// Vocabulary tiles a workgroup takes one after another, and such sweeps: the
// least time for rounds of 512 workgroups, which need about as long to begin as
// for 1.5 tiles.  us of the derivatives with sweeps of 2 and of 8 tiles (16,384
// tokens x 4,096 rows, width 256): 77 and 61.
void plan_sweeps(uint32_t ttiles, uint32_t vtiles, uint32_t &sweep, uint32_t &sweeps) {
  uint64_t best = ~0ull;
  const uint64_t most = 1u << 23;  // workgroups of a launch
  for (uint64_t s = 1; s <= vtiles; s = s < 64 ? s + 1 : 2 * s) {
    const uint64_t work = ttiles * host_ceil_div(vtiles, s),
                   cost = host_ceil_div(work, 512) * (2 * s + 3);
    if (s > 1 && (cost >= best || s > 64) && ttiles * host_ceil_div(vtiles, sweep) <= most) continue;
    best = cost;
    sweep = (uint32_t)s;
  }
  sweeps = (vtiles + sweep - 1) / sweep;
}

// Tiles of a call through registers: of 64 where those of 128 leave CUs without one
// or would be half empty.  us with tiles of 64 and of 128: loss of 30 tokens x 19,106
// rows x width 719 bfloat16 22 and 35; loss and gradient of 130 x 901 x 847 bfloat16
// 30 and 65, 1,000 x 4,096 x 64 float32 41 and 44, 46 x 241,327 x 79 bfloat16 154 and
// 169, 200 x 30,000 x 500 float32 254 and 207.
uint32_t staged_tile(uint64_t tokens, uint64_t rows) {
  return tokens <= 64 || host_ceil_div(tokens, 128) * host_ceil_div(rows, 128) <= 256 ? 64 : 128;
}

Tiling tiling(uint64_t tokens, uint64_t rows, uint32_t tile) {
  Tiling t = {};
  t.ttiles = (uint32_t)host_ceil_div(tokens, tile);
  t.vtiles = (uint32_t)host_ceil_div(rows, tile);
  if (t.vtiles) plan_sweeps(t.ttiles, t.vtiles, t.sweep, t.sweeps);
  return t;
}

constexpr uint32_t kPad = 256;  // of tokens and pieces: whole tiles of any kind

// How a call's tiles come to LDS: through registers; straight from its inputs,
// bfloat16 rows of whole 64s at 16-byte boundaries; or straight from copies of
// them in the workspace, bfloat16 rows padded with zeros, a piece of the vocabulary
// at a time.  Hangs on addresses too; the workspace has room for either way.
enum class Way { kStaged, kDirect, kPacked };

// Tiles of z of a call.
uint64_t whole_tiles(const nsfps_loss_args &a) {
  return host_ceil_div(a.tokens, kTile) * host_ceil_div(a.rows, kTile);
}
// Whether copies of the inputs pay for the loss.  us with and without, 5,003 rows:
// 512 tokens of width 847 29 and 34, 1,024 of 257 21 and 19, 8,192 of 65 31 and 35.
bool loss_packs(const nsfps_loss_args &a) {
  return a.dtype == NSFPS_BF16 && a.tokens >= 512 && a.rows >= kPad &&
         whole_tiles(a) * a.width >= 1u << 17;
}
// Whether the gradient's tiles go straight to LDS, from the inputs or their copies
// (tokens are padded to whole tiles there, and all tiles are of 128).  us of loss
// and gradient so and through registers, aligned: 256 tokens x 5,003 rows x width
// 256 39 and 33, 512 x 5,003 x 256 41 and 41, 1,024 x 5,003 x 256 48 and 51, 2,048
// x 1,024 x 1,024 74 and 70, 2,048 x 5,003 x 1,024 164 and 197; copied: 512 x 5,003
// x 257 49 and 53, 1,024 x 5,003 x 65 54 and 49, 8,192 x 5,003 x 847 420 and 532.
// (Three planes of a float32 call's terms, copied, lost by up to a quarter: the
// products of the terms bound it, not the loads.)
bool grad_straight(const nsfps_loss_args &a, bool one) {
  return one && a.tokens >= kPad && a.rows >= kPad && whole_tiles(a) > 128 &&
         whole_tiles(a) * a.width >= 40000;
}
bool direct_sizes(const nsfps_loss_args &a) {
  return a.dtype == NSFPS_BF16 && a.width % 64 == 0 && a.x_stride % 8 == 0 &&
         a.table_stride % 8 == 0 &&
         std::max(a.x_stride, a.table_stride) < 1u << 23;  // (a Feed's offsets)
}
bool direct_places(const nsfps_loss_args &a) {
  return ((uintptr_t)a.d_x | (uintptr_t)a.d_table) % 16 == 0;
}

LogitDev logits(const nsfps_loss_args &a, const Matrix &x, const Matrix &e, uint64_t row0,
                uint64_t x_rows, uint64_t e_rows, uint32_t tile) {
  LogitDev d = {};
  d.x = x;
  d.e = e;
  d.tiles = tiling(x_rows, e_rows, tile);
  d.scale2 = a.scale * kLog2e;
  d.to_2 = std::fabs(a.scale) < 1e-30f ? kLog2e : (double)d.scale2 / a.scale;
  d.row0 = (uint32_t)row0;
  d.lse = a.d_lse;
  return d;
}
// x and rows of the table as they are
Matrix x_of(const nsfps_loss_args &a) {
  return {a.d_x, a.x_stride, (uint32_t)a.tokens, a.width};
}
Matrix table_of(const nsfps_loss_args &a, uint64_t row0, uint64_t rows) {
  return {(const char *)a.d_table + row0 * a.table_stride * (a.dtype == NSFPS_F32 ? 4 : 2),
          a.table_stride, (uint32_t)rows, a.width};
}

// f(the walk of tiles straight to LDS).  Tokens in registers, which take their time
// to come there, pay in long sweeps.  us of the loss with and without, width 256:
// 16,384 tokens x 16,384 rows (sweeps of 32 tiles) 141 and 164, x 4,096 (8) 50 and
// 51, x 2,048 (4) 35 and 32, 4,096 x 2,048 (1) 20 and 14; width 128, 16,384 tokens
// x 4,096 rows 32 and 34, x 2,048 22 and 22, x 1,024 (2) 18 and 15.
template <typename F>
void by_steps(uint32_t width, uint32_t sweep, F f) {
  if (sweep < 8) return f(DirectLogits());
  switch (width) {
    case 64: return f(ResidentLogits<64, 1>());
    case 128: return f(ResidentLogits<128, 1>());
    case 192: return f(ResidentLogits<64, 3>());
    case 256: return f(ResidentLogits<128, 2>());
    default: return f(DirectLogits());
  }
}

template <Ends kEnds>
using EndsOf = std::integral_constant<Ends, kEnds>;
template <typename F>
void by_ends(uint32_t width, uint32_t tile, F f) {
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, 4> four;
  if (width < 8)
    tile == 64 ? f(EndsOf<Ends::kNarrow>(), two) : f(EndsOf<Ends::kNarrow>(), four);
  else
    tile == 64 ? f(EndsOf<Ends::kWide>(), two) : f(EndsOf<Ends::kWide>(), four);
}

template <typename Logits>
hipError_t run_stats(const LogitDev &d, hipStream_t st) {
  k_loss_stats<Logits><<<xcd_grid((uint64_t)d.tiles.ttiles * d.tiles.sweeps), 256, 0, st>>>(d);
  return hipGetLastError();
}
template <typename Logits, typename D>
hipError_t run_d(const LogitDev &d, hipStream_t st) {
  k_loss_d<Logits, D><<<xcd_grid((uint64_t)d.tiles.ttiles * d.tiles.sweeps), 256, 0, st>>>(d);
  return hipGetLastError();
}
template <int WM, int WN, int MT>
hipError_t run_direct(const ProductDev &dx, const ProductDev &de, uint32_t grid, hipStream_t st) {
  typedef DirectProduct<WM, WN, MT, false> X;
  const size_t lds = sizeof(typename X::Lds);
  static_assert(sizeof(typename X::Lds) == sizeof(typename DirectProduct<WM, WN, MT, true>::Lds), "LDS");
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void *)k_loss_products_direct<WM, WN, MT>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  k_loss_products_direct<WM, WN, MT><<<grid, 64 * WM * WN, lds, st>>>(dx, de);
  return hipGetLastError();
}

// The copy that a PackDev makes; and one or two of them in a launch.
Matrix packed(const PackDev &p) {
  return {p.out, p.out_cols, (uint32_t)p.out_rows, p.out_cols};
}
hipError_t run_pack(const PackDev &first, const PackDev *second, hipStream_t st) {
  const auto threads = [](const PackDev &p) { return p.out_rows * (p.out_cols / 8); };
  const uint32_t grid = grid_of(std::max(threads(first), second ? threads(*second) : 0));
  k_loss_pack<<<dim3(grid, second ? 2 : 1), 256, 0, st>>>(first, second ? *second : first);
  return hipGetLastError();
}

// The sums of one product, or of two, as rows of their results.  A group of lanes
// takes a value where results are too few to fill the chip (46 tokens x 241,327 rows
// x width 79, 512 splits: 6 us, 30 with a lane a value).
hipError_t write_out(ProductDev first, const ProductDev *other, hipStream_t st) {
  ProductDev second = other ? *other : first;
  const auto threads = [](ProductDev &d) {
    const uint64_t values = (uint64_t)d.out_rows * ((d.out_cols + 3) / 4);
    d.out_lanes = 1;
    while (d.out_lanes < 64 && 8 * d.out_lanes < d.splits && values * d.out_lanes < 1u << 17)
      d.out_lanes *= 2;
    return values * d.out_lanes;
  };
  const uint32_t grid = grid_of(std::max(threads(first), threads(second)));
  k_loss_out<<<dim3(grid, other ? 2 : 1), 256, 0, st>>>(first, second);
  return hipGetLastError();
}

hipError_t write_zeros(uint32_t dtype, void *out, uint64_t stride, uint64_t rows, uint32_t width,
                       hipStream_t st) {
  if (!rows) return hipSuccess;
  if (dtype == NSFPS_F32)
    k_loss_zeros<float><<<grid_of(rows * width), 256, 0, st>>>((float *)out, stride, rows, width);
  else
    k_loss_zeros<bf16><<<grid_of(rows * width), 256, 0, st>>>((bf16 *)out, stride, rows, width);
  return hipGetLastError();
}

#define LAUNCH(expr)                      \
  do {                                    \
    const hipError_t e_ = (expr);         \
    if (e_ != hipSuccess) return e_;      \
  } while (0)

// Places in a workspace.
struct Places {
  uint64_t at = 0;
  uint64_t take(uint64_t n) {
    const uint64_t was = at;
    at += bytes256(n);
    return was;
  }
};

struct LossPlan {
  Way way;
  uint32_t tile, width;  // of packed rows
  uint64_t piece, pieces, nparts;  // rows of a piece; parts of all pieces
  uint64_t parts, x, e, bytes;
};
LossPlan loss_plan(const nsfps_loss_args &a, Way way) {
  LossPlan p = {};
  p.way = way;
  p.tile = way == Way::kStaged ? staged_tile(a.tokens, a.rows) : kTile;
  p.width = (uint32_t)up(a.width, 64);
  p.piece = way == Way::kPacked ? std::min<uint64_t>(a.rows, 1u << 16) : a.rows;
  p.pieces = a.rows ? host_ceil_div(a.rows, p.piece) : 0;
  for (uint64_t k = 0; k < std::min<uint64_t>(p.pieces, 2); ++k) {  // whole pieces, and the last
    const uint64_t rows = k ? a.rows - (p.pieces - 1) * p.piece : p.piece,
                   sweeps = tiling(a.tokens, rows, p.tile).sweeps;
    p.nparts += k ? sweeps : p.pieces > 1 ? (p.pieces - 1) * sweeps : sweeps;
  }
  Places w;
  p.parts = w.take(8 * p.nparts * up(a.tokens, 16));
  if (way == Way::kPacked) {
    p.x = w.take(2ull * a.tokens * p.width);
    p.e = w.take(2ull * p.piece * p.width);
  }
  p.bytes = std::max<uint64_t>(256, w.at);
  return p;
}
Way loss_fallback(const nsfps_loss_args &a) {
  return loss_packs(a) ? Way::kPacked : Way::kStaged;
}

struct GradPlan {
  Way way;
  uint64_t tokens;             // padded
  uint64_t piece, pieces;      // vocabulary rows of a piece, a multiple of kPad
  uint32_t mt, nt;             // rows and columns of a product's tile
  uint32_t width;              // of packed rows
  uint32_t per, dx_splits, de_splits;
  uint64_t d_size, d_ld;       // (rows a whole number of 4 KB apart meet in one memory channel)
  bool dx_sums, de_sums;
  uint64_t x, e, d, dx, de, bytes;  // workspace offsets
};

// k of a split, of both products alike.  at_once workgroups run at once and take 1
// us for 64 terms of a pass; splits' sums go to memory and come back, 4 TB/s.  The
// split with the least of both.  us of the products of 16,384 tokens and pieces of
// 4,096 rows, width 383 in float32: 620 so, 888 with as many splits as just fill
// the chip.  No split of fewer than 256 terms: loss and gradient of 30 tokens x
// 19,106 rows x width 719 bfloat16 69, 77 with 128.
void plan_splits(GradPlan &p, uint64_t dx_tiles, uint64_t dx_terms, uint64_t de_tiles,
                 uint64_t de_terms, uint32_t passes, uint64_t at_once, uint64_t dx_bytes,
                 uint64_t de_bytes) {
  double best = 0.;
  for (uint64_t n = 1; n <= 512; ++n) {
    const uint64_t per = up(host_ceil_div(std::max(dx_terms, de_terms), n), 64);
    if (n > 1 && per < 256) break;
    const uint64_t dx = host_ceil_div(dx_terms, per), de = host_ceil_div(de_terms, per);
    const double rounds = (double)host_ceil_div(dx_tiles * dx + de_tiles * de, at_once);
    const double longest = (double)std::min(per, std::max(dx_terms, de_terms));
    const double sums = (dx > 1 || p.pieces > 1 ? 2. * dx * dx_bytes : 0.) +
                        (de > 1 ? 2. * de * de_bytes : 0.);
    const double us = rounds * longest / 64. * passes + sums / 4e6;
    if (n == 1 || us < best) {
      best = us;
      p.per = (uint32_t)per;
      p.dx_splits = (uint32_t)dx;
      p.de_splits = (uint32_t)de;
    }
  }
}

GradPlan grad_plan(const nsfps_loss_args &a, uint32_t grad_dtype, Way way) {
  GradPlan p = {};
  p.way = way;
  p.tokens = up(a.tokens, kPad);
  const uint64_t whole = up(a.rows, kPad);
  p.bytes = 256;
  if (!p.tokens || !whole) return p;
  const bool one = a.dtype == NSFPS_BF16 && grad_dtype == NSFPS_BF16, direct = way != Way::kStaged;
  p.width = (uint32_t)up(a.width, 64);
  p.d_size = one ? 2 : 4;
  // a piece of d: 64 million values, and 1,024 rows at least
  constexpr uint64_t kValues = 1ull << 26;
  p.piece = std::min(whole, std::max<uint64_t>(1024, kValues / p.tokens / kPad * kPad));
  p.pieces = host_ceil_div(whole, p.piece);
  // columns: us of 8,192 x 5,003 x 256 bfloat16 140, 142 with 128; of 16,384 x 8,192
  // x 64 float32 521, 632 with 128
  if (direct) {
    p.nt = p.width % 256 == 0 ? 256 : p.width % 128 == 0 ? 128 : 64;
    p.mt = p.nt < 256 ? 256 : kTile;
  } else {
    p.nt = a.width <= 64 ? 64 : 128;
    p.mt = kTile;
  }
  const uint64_t ntiles = host_ceil_div(a.width, p.nt), ld = ntiles * p.nt;
  plan_splits(p, p.tokens / p.mt * ntiles, std::min(p.piece, a.rows), p.piece / p.mt * ntiles,
              a.tokens, a.dtype == NSFPS_F32 ? 6 : one ? 1 : 2, direct ? 256 : 512,
              4 * a.tokens * ld, 4 * p.piece * ld);
  p.dx_sums = p.dx_splits > 1 || p.pieces > 1;
  p.de_sums = p.de_splits > 1;
  Places w;
  if (direct) p.x = w.take(2ull * p.tokens * p.width);
  if (way == Way::kPacked) p.e = w.take(2ull * p.piece * p.width);
  p.d_ld = p.piece + 256 / p.d_size;
  p.d = w.take(p.d_size * p.tokens * p.d_ld);
  p.dx = w.take(p.dx_sums ? 4 * p.dx_splits * a.tokens * ld : 0);
  p.de = w.take(p.de_sums ? 4 * p.de_splits * p.piece * ld : 0);
  p.bytes = w.at;
  return p;
}
Way grad_way(const nsfps_loss_args &a, bool one, bool direct) {
  return !grad_straight(a, one) ? Way::kStaged : direct ? Way::kDirect : Way::kPacked;
}

}  // namespace

uint64_t loss_bytes(const nsfps_loss_args &a) {
  const uint64_t other = loss_plan(a, loss_fallback(a)).bytes;
  return direct_sizes(a) ? std::max(other, loss_plan(a, Way::kDirect).bytes) : other;
}

hipError_t launch_loss(const nsfps_loss_args &a, hipStream_t st) {
  const Way way = direct_sizes(a) && direct_places(a) ? Way::kDirect : loss_fallback(a);
  const LossPlan p = loss_plan(a, way);
  char *const ws = (char *)a.workspace;
  const uint64_t stride = up(a.tokens, 16);
  Matrix x = x_of(a);
  const PackDev px = {x, nullptr, 0, p.width, (bf16 *)(ws + p.x), a.tokens};
  if (way == Way::kPacked) x = packed(px);
  float2 *parts = (float2 *)(ws + p.parts);
  for (uint64_t k = 0; k < p.pieces; ++k) {
    const uint64_t row0 = k * p.piece, rows = std::min(p.piece, a.rows - row0);
    Matrix e = table_of(a, row0, rows);
    if (way == Way::kPacked) {
      const PackDev pe = {e, nullptr, 0, p.width, (bf16 *)(ws + p.e), rows};
      LAUNCH(run_pack(pe, k ? nullptr : &px, st));
      e = packed(pe);
    }
    LogitDev d = logits(a, x, e, row0, a.tokens, rows, p.tile);
    d.parts = parts;
    d.part_stride = stride;
    parts += d.tiles.sweeps * stride;
    hipError_t rc = hipSuccess;
    const auto go = [&](auto z) { rc = run_stats<decltype(z)>(d, st); };
    if (way != Way::kStaged)
      by_steps(p.width, d.tiles.sweep, go);
    else
      by_ends(a.width, p.tile, [&](auto ends, auto tiles) {
        constexpr Ends kEnds = decltype(ends)::value;
        constexpr int kTiles = decltype(tiles)::value;
        a.dtype == NSFPS_F32 ? go(StagedLogits<float, 3, false, kEnds, kTiles>())
                             : go(StagedLogits<bf16, 1, true, kEnds, kTiles>());
      });
    LAUNCH(rc);
  }
  const double to_e = std::fabs((double)a.scale) / exponent_by(a.scale * kLog2e);
  const auto join = [&](auto t) {
    // as many workgroups as fill the chip (us of 7 tokens x 262,144 rows 30, 46 with
    // 16 tokens a workgroup; with gradient 16,384 x 8,192 x 64 220, 235 with one)
    uint32_t group = 16;
    while (group > 1 && a.tokens / group < 256) group /= 2;
    const uint32_t grid = (uint32_t)std::min<uint64_t>(1u << 16, host_ceil_div(a.tokens, group));
    k_loss_join<decltype(t)><<<grid, 256, 0, st>>>(
        (const float2 *)(ws + p.parts), (uint32_t)p.nparts, stride, group, x_of(a),
        table_of(a, 0, a.rows), a.scale, to_e, a.d_targets, a.d_loss, a.d_lse);
    return hipGetLastError();
  };
  return a.dtype == NSFPS_F32 ? join(float()) : join(bf16());
}

uint64_t loss_grad_bytes(const nsfps_loss_args &a, const nsfps_loss_grads &g) {
  const bool one = a.dtype == NSFPS_BF16 && g.grad_dtype == NSFPS_BF16;
  return grad_plan(a, g.grad_dtype, grad_way(a, one, false)).bytes;  // (the copies' is the larger)
}

hipError_t launch_loss_grad(const nsfps_loss_args &a, const nsfps_loss_grads &g, hipStream_t st) {
  const bool one = a.dtype == NSFPS_BF16 && g.grad_dtype == NSFPS_BF16;
  const Way way = grad_way(a, one, direct_sizes(a) && direct_places(a));
  const bool direct = way != Way::kStaged;
  const GradPlan p = grad_plan(a, g.grad_dtype, way);
  if (!p.pieces) {
    LAUNCH(write_zeros(a.dtype, g.d_dx, g.dx_stride, a.tokens, a.width, st));
    return write_zeros(g.grad_dtype, g.d_dtable, g.dtable_stride, a.rows, a.width, st);
  }
  char *const ws = (char *)a.workspace;
  const uint32_t ntiles = (uint32_t)host_ceil_div(a.width, p.nt);
  const uint64_t z = g.grad_dtype == NSFPS_F32 ? 4 : 2;
  Matrix x = x_of(a);
  // whole tiles, and zeros for rows that count for nothing
  const PackDev px = {x, a.d_targets, (uint32_t)a.rows, p.width, (bf16 *)(ws + p.x), p.tokens};
  if (way == Way::kDirect) LAUNCH(run_pack(px, nullptr, st));
  if (direct) x = packed(px);
  ProductDev dx = {};
  dx.weights = {g.d_dloss, a.d_targets, (uint32_t)a.tokens, (uint32_t)a.rows, a.scale};
  dx.mtiles = (uint32_t)host_ceil_div(a.tokens, p.mt);
  dx.ntiles = ntiles;
  dx.per = p.per;
  dx.out = g.d_dx;
  dx.out_ld = g.dx_stride;
  dx.out_rows = (uint32_t)a.tokens;
  dx.out_cols = a.width;
  dx.out_dtype = a.dtype;
  dx.sums = p.dx_sums ? (float *)(ws + p.dx) : nullptr;
  dx.sums_ld = (uint64_t)ntiles * p.nt;
  dx.sums_split = a.tokens * dx.sums_ld;
  for (uint64_t k = 0; k < p.pieces; ++k) {
    const uint64_t row0 = k * p.piece, rows = std::min(p.piece, a.rows - row0);
    Matrix e = table_of(a, row0, rows);
    if (way == Way::kPacked) {
      const PackDev pe = {e, nullptr, 0, p.width, (bf16 *)(ws + p.e), rows};
      LAUNCH(run_pack(pe, k ? nullptr : &px, st));
      e = packed(pe);
    }
    const uint32_t tile = direct ? kTile : staged_tile(a.tokens, rows);
    LogitDev l = direct ? logits(a, x, e, row0, p.tokens, up(rows, kPad), tile)
                        : logits(a, x, e, row0, a.tokens, rows, tile);
    l.weights = dx.weights;
    l.d = ws + p.d;
    l.d_ld = p.d_ld;
    hipError_t rc = hipSuccess;
    if (direct)
      by_steps(p.width, l.tiles.sweep, [&](auto w) { rc = run_d<decltype(w), bf16>(l, st); });
    else
      by_ends(a.width, tile, [&](auto ends, auto tiles) {
        constexpr Ends kEnds = decltype(ends)::value;
        constexpr int kTiles = decltype(tiles)::value;
        rc = a.dtype == NSFPS_F32 ? run_d<StagedLogits<float, 3, false, kEnds, kTiles>, float>(l, st)
             : one ? run_d<StagedLogits<bf16, 1, true, kEnds, kTiles>, bf16>(l, st)
                   : run_d<StagedLogits<bf16, 1, false, kEnds, kTiles>, float>(l, st);
      });
    LAUNCH(rc);

    dx.m = {ws + p.d, p.d_ld, (uint32_t)(direct ? p.tokens : a.tokens), (uint32_t)rows};
    dx.n = e;
    dx.terms = (uint32_t)rows;
    dx.splits = p.dx_splits;  // those of a short last piece may be empty: they add nothing
    dx.add = k > 0;
    ProductDev de = dx;
    de.n = x;
    de.mtiles = (uint32_t)host_ceil_div(rows, p.mt);
    de.terms = (uint32_t)a.tokens;
    de.splits = p.de_splits;
    de.out = (char *)g.d_dtable + row0 * g.dtable_stride * z;
    de.out_ld = g.dtable_stride;
    de.out_rows = (uint32_t)rows;
    de.out_dtype = g.grad_dtype;
    de.sums = p.de_sums ? (float *)(ws + p.de) : nullptr;
    de.sums_split = p.piece * de.sums_ld;
    de.add = 0;
    const uint32_t work = xcd_grid((uint64_t)dx.mtiles * ntiles * dx.splits +
                                   (uint64_t)de.mtiles * ntiles * de.splits);
    const auto staged = [&](auto nt, auto ends) {
      constexpr int NT = decltype(nt)::value;
      constexpr Ends kEnds = decltype(ends)::value;
      if (a.dtype == NSFPS_F32)
        k_loss_products<float, 3, 3, float, 3, NT, kEnds><<<work, 256, 0, st>>>(dx, de);
      else if (one)
        k_loss_products<bf16, 1, 1, bf16, 1, NT, kEnds><<<work, 256, 0, st>>>(dx, de);
      else
        k_loss_products<float, 1, 2, bf16, 1, NT, kEnds><<<work, 256, 0, st>>>(dx, de);
      return hipGetLastError();
    };
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 4> four;
    if (direct)
      rc = p.nt == 256   ? run_direct<2, 4, 4>(dx, de, work, st)
           : p.nt == 128 ? run_direct<4, 2, 4>(dx, de, work, st)
                         : run_direct<4, 1, 4>(dx, de, work, st);
    else
      rc = a.width < 8   ? staged(two, EndsOf<Ends::kNarrow>())
           : p.nt == 64 ? staged(two, EndsOf<Ends::kWide>())
                        : staged(four, EndsOf<Ends::kWide>());
    LAUNCH(rc);
    const bool last = k + 1 == p.pieces;
    if (de.sums) LAUNCH(write_out(de, last && dx.sums ? &dx : nullptr, st));
    if (!de.sums && last && dx.sums) LAUNCH(write_out(dx, nullptr, st));
  }
  return hipSuccess;
}

hipError_t preload_loss_kernels() {
  return func_attributes(k_loss_stats<ResidentLogits<128, 2>>, k_loss_join<bf16>,
                         k_loss_d<ResidentLogits<128, 2>, bf16>, k_loss_products_direct<2, 4, 4>,
                         k_loss_out, k_loss_pack);
}

}  // namespace nsfps
