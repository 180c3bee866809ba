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
#include "nsfps_launch.h"
#include "nsfps_product.h"

#include <algorithm>
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

// ---- tiles of z

struct LogitDev {
  Matrix x, e;                // e: the piece
  uint32_t ttiles, vtiles;    // tiles of tokens, of the piece's vocabulary
  uint32_t sweep, sweeps;     // vocabulary tiles a workgroup takes one after another
  float scale2;               // scale * log2(e)
  // statistics
  float2 *parts;              // [sweeps][part_stride]: maximum and sum, in powers of two
  uint64_t part_stride;
  // gradient
  const float *lse, *dloss;
  const int32_t *targets;
  uint32_t row0, vocabulary;  // the piece's first row, rows of the whole table
  float scale;
  void *d;                    // [tokens][d_ld] (kDirect: whole tiles of tokens)
  uint64_t d_ld;
};

// Workgroup w's tile of tokens and sweep: tokens change fastest, within groups
// that share sweeps, so that workgroups of one XCD read the same rows.
__device__ __forceinline__ bool logit_item(const LogitDev &a, uint32_t &ttile, uint32_t &first,
                                           uint32_t &last) {
  const uint32_t work = a.ttiles * a.sweeps, per = (work + 7) / 8;
  const uint32_t w = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || w >= work) return false;
  constexpr uint32_t kGroup = 8;
  const uint32_t whole = kGroup * a.sweeps, group = w / whole, t0 = group * kGroup;
  const uint32_t size = min(kGroup, a.ttiles - t0), in = w - group * whole;
  ttile = t0 + in % size;
  first = in / size * a.sweep;
  last = min(first + a.sweep, a.vtiles);
  return true;
}

// The tiles of z that a workgroup walks, one after another; epilogue(sum, tile)
// has each.  Operands through registers: any rows, either type.
template <typename T, int P>
struct StagedLogits {
  static constexpr int kTerms = P == 1 ? 64 : 32;
  typedef Product<2, 2, 4, 4, kTerms, P, P, false, false, true> Prod;
  typedef typename Prod::Lds Lds;
  static constexpr bool kDirect = false;

  template <typename F>
  static __device__ __forceinline__ void walk(const LogitDev &a, Lds &lds, uint32_t ttile,
                                              uint32_t first, uint32_t last, F epilogue) {
    Stage<T, kTile, kTerms, 256> sx, se;
    const uint32_t width = a.x.cols, steps = ceil_div(width, kTerms);
    const uint32_t t0 = ttile * kTile;
    const T *const x = (const T *)a.x.p + (uint64_t)t0 * a.x.ld;
    const auto all = [](uint32_t) { return true; };
    uint32_t tile = first, k = 0;  // of the stage fetched next
    const auto fetch = [&] {
      const uint32_t v0 = tile * kTile;
      sx.fetch(x + k * kTerms, a.x.ld, a.x.rows - t0, width - k * kTerms, all);
      se.fetch((const T *)a.e.p + (uint64_t)v0 * a.e.ld + k * kTerms, a.e.ld, a.e.rows - v0,
               width - k * kTerms, all);
      if (++k == steps) k = 0, ++tile;
    };
    fetch();
    for (uint32_t t = first; t < last; ++t) {
      typename Prod::Sum sum = {};
      for (uint32_t s = 0; s < steps; ++s) {
        __syncthreads();
        sx.template put<Prod::kM, kTerms, false, P>(lds.m, Prod::kMPlane);
        se.template put<Prod::kN, kTerms, false, P>(lds.n, Prod::kNPlane);
        __syncthreads();
        if (tile < last) fetch();
        Prod::add(sum, lds);
      }
      epilogue(sum, t);
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

  template <typename F>
  static __device__ __forceinline__ void walk(const LogitDev &a, Lds &lds, uint32_t ttile,
                                              uint32_t first, uint32_t last, F epilogue) {
    Feed<kTile, 64, false, 256> fx, fe;
    const uint32_t steps = a.x.cols / 64;
    fx.start((const bf16 *)a.x.p + (uint64_t)ttile * kTile * a.x.ld, a.x.ld,
             a.x.rows - ttile * kTile);
    uint32_t tile = first, k = 0, buf = 0;  // of the stage issued next
    const auto issue = [&](uint32_t b) {
      if (k == 0)
        fe.start((const bf16 *)a.e.p + (uint64_t)tile * kTile * a.e.ld, a.e.ld,
                 a.e.rows - tile * kTile);
      fx.issue(lds.buf[b].m, 64 * k);
      fe.issue(lds.buf[b].n, 64 * k);
      if (++k == steps) k = 0, ++tile;
    };
    issue(0);
    for (uint32_t t = first; t < last; ++t) {
      typename Prod::Sum sum = {};
      for (uint32_t s = 0; s < steps; ++s) {
        wait_loads();
        __syncthreads();
        Prod::add_then(sum, lds.buf[buf], [&] {
          if (tile < last) issue(buf ^ 1);
        });
        buf ^= 1;
      }
      epilogue(sum, t);
    }
  }
};

__device__ __forceinline__ void join_stats(float &m, float &s, float m2, float s2) {
  const float top = fmaxf(m, m2), at = top == -INFINITY ? 0.f : top;
  s = s * exp2_fast(m - at) + s2 * exp2_fast(m2 - at);
  m = top;
}

template <typename Logits>
__global__ __launch_bounds__(256, 2) void k_loss_stats(LogitDev a) {
  __shared__ typename Logits::Lds lds;
  __shared__ float2 s_part[2][kTile];
  uint32_t ttile, first, last;
  if (!logit_item(a, ttile, first, last)) return;
  const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / 2, wn = wave % 2;
  float top[4], sum[4];  // of this lane's columns, for its four tokens
#pragma unroll
  for (int i = 0; i < 4; ++i) top[i] = -INFINITY, sum[i] = 0.f;
  Logits::walk(a, lds, ttile, first, last, [&](f32x4(&z)[4][4], uint32_t tile) {
    const uint32_t v0 = tile * kTile + 64 * wn + 16 * g;
    const bool ragged = (tile + 1) * kTile > a.e.rows;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float m = top[i];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v = z[i][j][r] * a.scale2;
          if (ragged && v0 + 4 * j + r >= a.e.rows) v = -INFINITY;
          z[i][j][r] = v;
          m = fmaxf(m, v);
        }
      const float at = m == -INFINITY ? 0.f : m;
      float s = sum[i] * exp2_fast(top[i] - at);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s += exp2_fast(z[i][j][r] - at);
      top[i] = m;
      sum[i] = s;
    }
  });
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int off = 16; off < 64; off <<= 1)
      join_stats(top[i], sum[i], __shfl_xor(top[i], off, 64), __shfl_xor(sum[i], off, 64));
    if (g == 0) s_part[wn][64 * wm + 16 * i + l] = make_float2(top[i], sum[i]);
  }
  __syncthreads();
  const uint32_t token = ttile * kTile + threadIdx.x;
  if (threadIdx.x < kTile && token < a.x.rows) {
    float2 v = s_part[0][threadIdx.x];
    join_stats(v.x, v.y, s_part[1][threadIdx.x].x, s_part[1][threadIdx.x].y);
    a.parts[first / a.sweep * a.part_stride + token] = v;
  }
}

// lse and loss of 16 tokens: 16 runs of parts each, then a wave finds the
// logits of four tokens' targets.
template <typename T>
__global__ __launch_bounds__(256) void k_loss_join(const float2 *__restrict__ parts, uint32_t nparts,
                                                   uint64_t part_stride, Matrix x, Matrix table,
                                                   float scale, const int32_t *__restrict__ targets,
                                                   float *__restrict__ loss,
                                                   float *__restrict__ lse) {
  __shared__ float2 s_part[4][16];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, tokens = x.rows;
  for (uint32_t t0 = blockIdx.x * 16; t0 < tokens; t0 += gridDim.x * 16) {
    const uint32_t mine = min(t0 + lane % 16, tokens - 1);
    float m = -INFINITY, s = 0.f;
    for (uint32_t p = threadIdx.x / 16; p < nparts; p += 16) {
      const float2 v = parts[p * part_stride + mine];
      join_stats(m, s, v.x, v.y);
    }
#pragma unroll
    for (int off = 16; off < 64; off <<= 1)
      join_stats(m, s, __shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
    if (lane < 16) s_part[wave][lane] = make_float2(m, s);
    float dot[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t token = t0 + 4 * wave + i;
      dot[i] = 0.f;
      if (token < tokens && (uint32_t)targets[token] < table.rows) {
        const T *xr = (const T *)x.p + token * x.ld,
                *er = (const T *)table.p + (uint64_t)(uint32_t)targets[token] * table.ld;
        for (uint32_t c = lane; c < x.cols; c += 64) {
          float u[1], v[1];
          load_f32<T, 1>(xr + c, u);
          load_f32<T, 1>(er + c, v);
          dot[i] = fmaf(u[0], v[0], dot[i]);
        }
      }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) dot[i] += __shfl_xor(dot[i], off, 64);
    __syncthreads();
    const uint32_t token = t0 + 4 * wave + lane;
    if (lane < 4 && token < tokens) {
      float2 v = s_part[0][4 * wave + lane];
#pragma unroll
      for (int k = 1; k < 4; ++k)
        join_stats(v.x, v.y, s_part[k][4 * wave + lane].x, s_part[k][4 * wave + lane].y);
      const float z = scale * (lane == 0 ? dot[0] : lane == 1 ? dot[1] : lane == 2 ? dot[2] : dot[3]);
      const float all = (v.x + log2f(v.y)) * kLn2;
      lse[token] = all;
      loss[token] = (uint32_t)targets[token] < table.rows ? all - z : 0.f;
    }
    __syncthreads();
  }
}

// A piece's d, as D.
template <typename Logits, typename D>
__global__ __launch_bounds__(256, 2) void k_loss_d(LogitDev a) {
  __shared__ typename Logits::Lds lds;
  uint32_t ttile, first, last;
  if (!logit_item(a, ttile, first, last)) return;
  const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / 2, wn = wave % 2;
  const uint32_t token0 = ttile * kTile + 64 * wm + l;
  float lse2[4], weight[4];
  uint32_t target[4];  // in the piece
  bool counts[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t token = token0 + 16 * i;
    lse2[i] = weight[i] = 0.f;
    target[i] = ~0u;
    counts[i] = token < a.x.rows && (uint32_t)a.targets[token] < a.vocabulary;
    if (counts[i]) {
      lse2[i] = a.lse[token] * kLog2e;
      weight[i] = a.dloss[token] * a.scale;
      target[i] = (uint32_t)a.targets[token] - a.row0;
    }
  }
  Logits::walk(a, lds, ttile, first, last, [&](f32x4(&z)[4][4], uint32_t tile) {
    const uint32_t v0 = tile * kTile + 64 * wn + 16 * g;
    const bool ragged = (tile + 1) * kTile > a.e.rows;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t hit = target[i] - v0;
      float d[16];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p = exp2_fast(fmaf(z[i][j][r], a.scale2, -lse2[i]));
          if (hit == 4 * j + r) p -= 1.f;
          const bool in = counts[i] && (!ragged || v0 + 4 * j + r < a.e.rows);
          d[4 * j + r] = in ? p * weight[i] : 0.f;
        }
      if (!Logits::kDirect && token0 + 16 * i >= a.x.rows) continue;
      D *const out = (D *)a.d + (uint64_t)(token0 + 16 * i) * a.d_ld + v0;
      constexpr int V = kWide<D>;
#pragma unroll
      for (int k = 0; k < 16; k += V) {
        float o[V];
#pragma unroll
        for (int q = 0; q < V; ++q) o[q] = d[k + q];
        store_f32<D, V>(out + k, o);
      }
    }
  });
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
  uint32_t out_rows, out_cols, out_dtype, out_wide;  // wide: four values a store
  float *sums;           // [splits][rows][sums_ld], null: out is written
  uint64_t sums_split, sums_ld;
  uint32_t add;          // to what sums holds
  const int32_t *targets;  // of n's rows, null: all count
  uint32_t vocabulary;
};

template <typename Prod>
__device__ __forceinline__ void put_result(const ProductDev &a, const typename Prod::Sum &sum,
                                           uint32_t m0, uint32_t n0, uint32_t split) {
  constexpr int MT = sizeof(sum) / sizeof(sum[0]), NT = sizeof(sum[0]) / sizeof(sum[0][0]);
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
      const float v[4] = {sum[i][j][0], sum[i][j][1], sum[i][j][2], sum[i][j][3]};
      const auto store = [&](auto t) {
        using T = decltype(t);
        T *const out = (T *)a.out + row * a.out_ld + col;
        if (a.out_wide) {
          store_f32<T, 4>(out, v);
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
template <typename TM, int PM, typename TN, int PN, int NT, bool kMCol>
struct StagedProduct {
  static constexpr int kTerms = PM * PN == 1 ? 64 : 32;
  typedef Product<2, 2, 4, NT, kTerms, PM, PN, kMCol, true, false> Prod;
  static constexpr int kMRows = kMCol ? kTerms : Prod::kM, kMCols = kMCol ? Prod::kM : kTerms;

  static __device__ __forceinline__ void run(const ProductDev &a, typename Prod::Lds &lds,
                                             uint32_t w) {
    const ProductItem it = product_item(a, w);
    const uint32_t m0 = it.mt * Prod::kM, n0 = it.nt * Prod::kN;
    Stage<TM, kMRows, kMCols, 256> sm;
    Stage<TN, kTerms, Prod::kN, 256> sn;
    uint32_t k = it.k0;
    const auto fetch = [&] {
      const uint32_t mr = kMCol ? k : m0, mc = kMCol ? m0 : k;
      sm.fetch((const TM *)a.m.p + (uint64_t)mr * a.m.ld + mc, a.m.ld,
               (kMCol ? a.terms : a.m.rows) - mr, (kMCol ? a.m.cols : a.terms) - mc,
               [](uint32_t) { return true; });
      sn.fetch((const TN *)a.n.p + (uint64_t)k * a.n.ld + n0, a.n.ld, a.terms - k, a.n.cols - n0,
               [&](uint32_t r) {
                 return !a.targets || (uint32_t)a.targets[min(k + r, a.terms - 1)] < a.vocabulary;
               });
      k += kTerms;
    };
    typename Prod::Sum sum = {};
    if (it.k0 < it.k1) fetch();
    for (uint32_t s = it.k0; s < it.k1; s += kTerms) {
      __syncthreads();
      sm.template put<Prod::kM, kTerms, kMCol, PM>(lds.m, Prod::kMPlane);
      sn.template put<Prod::kN, kTerms, true, PN>(lds.n, Prod::kNPlane);
      __syncthreads();
      if (k < it.k1) fetch();
      Prod::add(sum, lds);
    }
    put_result<Prod>(a, sum, m0, n0, it.split);
  }
};

// Straight to LDS: bfloat16, M and N whole tiles (rows of N past its end are its
// last again, and meet zeros of M).
template <int NT, bool kMCol>
struct DirectProduct {
  typedef Product<2, 2, 4, NT, 64, 1, 1, kMCol, true, false> Prod;
  struct Lds {
    typename Prod::Lds buf[2];
  };

  static __device__ __forceinline__ void run(const ProductDev &a, Lds &lds, uint32_t w) {
    const ProductItem it = product_item(a, w);
    const uint32_t m0 = it.mt * Prod::kM, n0 = it.nt * Prod::kN;
    Feed<Prod::kM, 64, kMCol, 256> fm;
    Feed<Prod::kN, 64, true, 256> fn;
    const bf16 *const m = (const bf16 *)a.m.p + (kMCol ? m0 : (uint64_t)m0 * a.m.ld);
    const bf16 *const n = (const bf16 *)a.n.p + n0;
    fm.start(m, a.m.ld, ~0u);
    fn.start(n, a.n.ld, ~0u);
    uint32_t k = it.k0, buf = 0;
    const auto issue = [&](uint32_t b) {
      fm.issue(lds.buf[b].m, kMCol ? (uint64_t)k * a.m.ld : k);
      if (k + 64 > a.n.rows) {
        fn.start(n + (uint64_t)k * a.n.ld, a.n.ld, a.n.rows - k);
        fn.issue(lds.buf[b].n, 0);
      } else {
        fn.issue(lds.buf[b].n, (uint64_t)k * a.n.ld);
      }
      k += 64;
    };
    typename Prod::Sum sum = {};
    if (it.k0 < it.k1) issue(0);
    for (uint32_t s = it.k0; s < it.k1; s += 64) {
      wait_loads();
      __syncthreads();
      Prod::add_then(sum, lds.buf[buf], [&] {
        if (k < it.k1) issue(buf ^ 1);
      });
      buf ^= 1;
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

template <typename TD, int PDX, int PDE, typename T, int P, int NT>
__global__ __launch_bounds__(256, 2) void k_loss_products(ProductDev dx, ProductDev de) {
  typedef StagedProduct<TD, PDX, T, P, NT, false> X;
  typedef StagedProduct<TD, PDE, T, P, NT, true> E;
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
template <int NT>
__global__ __launch_bounds__(256, 2) void k_loss_products_direct(ProductDev dx, ProductDev de) {
  typedef DirectProduct<NT, false> X;
  typedef DirectProduct<NT, true> E;
  __shared__ union {
    typename X::Lds x;
    typename E::Lds e;
  } lds;
  uint32_t w;
  bool is_dx;
  if (!product_work(dx, de, w, is_dx)) return;
  if (is_dx)
    X::run(dx, lds.x, w);
  else
    E::run(de, lds.e, w);
}

// x as whole tiles of rows for the copies straight to LDS: zeros past the end
// and where a row counts for nothing, which may hold anything.
__global__ __launch_bounds__(256) void k_loss_rows(Matrix x, const int32_t *__restrict__ targets,
                                                   uint32_t vocabulary, bf16 *__restrict__ out,
                                                   uint64_t out_rows) {
  const uint32_t vecs = x.cols / 8;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < out_rows * vecs;
       i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = i / vecs, c = i % vecs * 8;
    u32x4 v = {0, 0, 0, 0};
    if (r < x.rows && (uint32_t)targets[r] < vocabulary)
      v = *(const NSFPS_GLOBAL_SEQ u32x4 *)((const bf16 *)x.p + r * x.ld + c);
    *(NSFPS_GLOBAL_SEQ u32x4 *)(out + r * x.cols + c) = v;
  }
}

// The splits' sums, added in order, as rows of the result.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_loss_out(ProductDev a) {
  const uint32_t vecs = (a.out_cols + V - 1) / V;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)a.out_rows * vecs;
       i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = i / vecs, c = i % vecs * V, at = r * a.sums_ld + c;
    float v[V] = {};
    for (uint32_t s = 0; s < a.splits; ++s) {
      float t[V];
      constexpr int W = V < 4 ? V : 4;
#pragma unroll
      for (int k = 0; k < V; k += W)
        load_f32<float, W>(a.sums + s * a.sums_split + at + k, *(float(*)[W])&t[k]);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] += t[k];
    }
    store_f32<T, V>((T *)a.out + r * a.out_ld + c, v);
  }
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

// Vocabulary tiles a workgroup takes one after another, and such sweeps: enough
// workgroups to fill the chip several times, few parts for each token.
void plan_sweeps(uint32_t ttiles, uint32_t vtiles, uint32_t &sweep, uint32_t &sweeps) {
  const uint64_t tiles = (uint64_t)ttiles * vtiles, most = 1u << 23;  // workgroups of a launch
  sweep = (uint32_t)std::max(std::min<uint64_t>({vtiles, 16, std::max<uint64_t>(1, tiles / 2048)}),
                             std::min<uint64_t>(vtiles, host_ceil_div(tiles, most)));
  sweeps = (vtiles + sweep - 1) / sweep;
}

struct LossPlan {
  uint32_t ttiles, vtiles, sweep, sweeps;
  uint64_t bytes;
};
LossPlan loss_plan(const nsfps_loss_args &a) {
  LossPlan p = {};
  p.ttiles = (uint32_t)host_ceil_div(a.tokens, kTile);
  p.vtiles = (uint32_t)host_ceil_div(a.rows, kTile);
  if (p.vtiles) plan_sweeps(p.ttiles, p.vtiles, p.sweep, p.sweeps);
  p.bytes = std::max<uint64_t>(256, bytes256(8 * p.sweeps * up(a.tokens, 16)));
  return p;
}

// kDirect of a call hangs on its addresses, the workspace does not: it has room
// for either.
struct GradPlan {
  uint64_t tokens;             // padded
  uint64_t piece, pieces;      // vocabulary rows of a piece, a multiple of kTile
  uint32_t nt;                 // columns of a product's tile
  uint32_t per, dx_splits, de_splits;
  uint64_t d_size;
  bool dx_sums, de_sums;
  uint64_t x, d, dx, de, bytes;  // workspace offsets
};
GradPlan grad_plan(const nsfps_loss_args &a, uint32_t grad_dtype) {
  GradPlan p = {};
  p.tokens = up(a.tokens, kTile);
  const uint64_t whole = up(a.rows, kTile);
  p.bytes = 256;
  if (!p.tokens || !whole) return p;
  const bool one = a.dtype == NSFPS_BF16 && grad_dtype == NSFPS_BF16;
  p.d_size = one ? 2 : 4;
  // a piece of d: 64 million values, and 1,024 rows at least
  constexpr uint64_t kValues = 1ull << 26;
  p.piece = std::min(whole, std::max<uint64_t>(1024, kValues / p.tokens / kTile * kTile));
  p.pieces = host_ceil_div(whole, p.piece);
  p.nt = a.width <= 64 ? 64 : 128;
  // k of a split: enough splits of both products to fill the chip
  const uint64_t ntiles = host_ceil_div(a.width, p.nt), dx_tiles = p.tokens / kTile * ntiles,
                 de_tiles = p.piece / kTile * ntiles,
                 dx_terms = std::min(p.piece, a.rows);
  constexpr uint64_t kFill = 512, kLeast = 256;
  p.per = (uint32_t)std::max(
      kLeast, up(host_ceil_div(dx_tiles * dx_terms + de_tiles * a.tokens, kFill), 64));
  p.dx_splits = (uint32_t)host_ceil_div(dx_terms, p.per);
  p.de_splits = (uint32_t)host_ceil_div(a.tokens, p.per);
  p.dx_sums = p.dx_splits > 1 || p.pieces > 1;
  p.de_sums = p.de_splits > 1;
  const uint64_t ld = ntiles * p.nt;
  uint64_t at = 0;
  const auto take = [&](uint64_t n) {
    const uint64_t was = at;
    at += bytes256(n);
    return was;
  };
  p.x = take(one ? 2 * p.tokens * a.width : 0);
  p.d = take(p.d_size * p.tokens * p.piece);
  p.dx = take(p.dx_sums ? 4 * p.dx_splits * a.tokens * ld : 0);
  p.de = take(p.de_sums ? 4 * p.de_splits * p.piece * ld : 0);
  p.bytes = at;
  return p;
}

// Whether tiles can go straight to LDS: bfloat16 rows of whole 64s at 16-byte
// boundaries.
bool direct_rows(const nsfps_loss_args &a) {
  return a.dtype == NSFPS_BF16 && a.width % 64 == 0 && a.x_stride % 8 == 0 &&
         a.table_stride % 8 == 0 && ((uintptr_t)a.d_x | (uintptr_t)a.d_table) % 16 == 0;
}

LogitDev logits(const nsfps_loss_args &a, uint64_t row0, uint64_t rows) {
  LogitDev d = {};
  const uint64_t size = a.dtype == NSFPS_F32 ? 4 : 2;
  d.x = {a.d_x, a.x_stride, (uint32_t)a.tokens, a.width};
  d.e = {(const char *)a.d_table + row0 * a.table_stride * size, a.table_stride, (uint32_t)rows,
         a.width};
  d.ttiles = (uint32_t)host_ceil_div(a.tokens, kTile);
  d.vtiles = (uint32_t)host_ceil_div(rows, kTile);
  plan_sweeps(d.ttiles, d.vtiles, d.sweep, d.sweeps);
  d.scale = a.scale;
  d.scale2 = a.scale * kLog2e;
  d.row0 = (uint32_t)row0;
  d.vocabulary = (uint32_t)a.rows;
  d.targets = a.d_targets;
  d.lse = a.d_lse;
  return d;
}

template <typename T>
bool wide_rows(const void *out, uint64_t ld, uint32_t width, uint32_t v) {
  return width % v == 0 && ld % v == 0 && (uintptr_t)out % (v * sizeof(T)) == 0;
}
bool wide_any(uint32_t dtype, const void *out, uint64_t ld, uint32_t width, uint32_t v) {
  return dtype == NSFPS_F32 ? wide_rows<float>(out, ld, width, v)
                            : wide_rows<bf16>(out, ld, width, v);
}

hipError_t write_out(const ProductDev &d, hipStream_t st) {
  const auto go = [&](auto t) {
    using T = decltype(t);
    constexpr int V = kWide<T>;
    if (wide_rows<T>(d.out, d.out_ld, d.out_cols, V))
      k_loss_out<T, V><<<grid_of((uint64_t)d.out_rows * (d.out_cols / V)), 256, 0, st>>>(d);
    else
      k_loss_out<T, 1><<<grid_of((uint64_t)d.out_rows * d.out_cols), 256, 0, st>>>(d);
    return hipGetLastError();
  };
  return d.out_dtype == NSFPS_F32 ? go(float()) : go(bf16());
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

}  // namespace

uint64_t loss_bytes(const nsfps_loss_args &a) { return loss_plan(a).bytes; }

hipError_t launch_loss(const nsfps_loss_args &a, hipStream_t st) {
  const LossPlan p = loss_plan(a);
  const uint64_t stride = up(a.tokens, 16);
  float2 *const parts = (float2 *)a.workspace;
  if (p.vtiles) {
    LogitDev d = logits(a, 0, a.rows);
    d.parts = parts;
    d.part_stride = stride;
    const uint32_t grid = xcd_grid((uint64_t)d.ttiles * d.sweeps);
    if (direct_rows(a))
      k_loss_stats<DirectLogits><<<grid, 256, 0, st>>>(d);
    else if (a.dtype == NSFPS_F32)
      k_loss_stats<StagedLogits<float, 3>><<<grid, 256, 0, st>>>(d);
    else
      k_loss_stats<StagedLogits<bf16, 1>><<<grid, 256, 0, st>>>(d);
    LAUNCH(hipGetLastError());
  }
  const auto join = [&](auto t) {
    k_loss_join<decltype(t)><<<grid_of(a.tokens * 16), 256, 0, st>>>(
        parts, p.sweeps, stride, Matrix{a.d_x, a.x_stride, (uint32_t)a.tokens, a.width},
        Matrix{a.d_table, a.table_stride, (uint32_t)a.rows, a.width}, a.scale, a.d_targets, a.d_loss,
        a.d_lse);
    return hipGetLastError();
  };
  return a.dtype == NSFPS_F32 ? join(float()) : join(bf16());
}

uint64_t loss_grad_bytes(const nsfps_loss_args &a, const nsfps_loss_grads &g) {
  return grad_plan(a, g.grad_dtype).bytes;
}

hipError_t launch_loss_grad(const nsfps_loss_args &a, const nsfps_loss_grads &g, hipStream_t st) {
  const GradPlan p = grad_plan(a, g.grad_dtype);
  if (!p.pieces) {
    LAUNCH(write_zeros(a.dtype, g.d_dx, g.dx_stride, a.tokens, a.width, st));
    return write_zeros(g.grad_dtype, g.d_dtable, g.dtable_stride, a.rows, a.width, st);
  }
  char *const ws = (char *)a.workspace;
  const bool one = p.d_size == 2, direct = one && direct_rows(a);
  const uint32_t ntiles = (uint32_t)host_ceil_div(a.width, p.nt);
  const uint64_t z = g.grad_dtype == NSFPS_F32 ? 4 : 2;
  const Matrix x = {a.d_x, a.x_stride, (uint32_t)a.tokens, a.width};
  if (direct) {
    k_loss_rows<<<grid_of(p.tokens * a.width / 8), 256, 0, st>>>(
        x, a.d_targets, (uint32_t)a.rows, (bf16 *)(ws + p.x), p.tokens);
    LAUNCH(hipGetLastError());
  }
  ProductDev dx = {};
  dx.mtiles = (uint32_t)(p.tokens / kTile);
  dx.ntiles = ntiles;
  dx.per = p.per;
  dx.out = g.d_dx;
  dx.out_ld = g.dx_stride;
  dx.out_rows = (uint32_t)a.tokens;
  dx.out_cols = a.width;
  dx.out_dtype = a.dtype;
  dx.out_wide = wide_any(a.dtype, g.d_dx, g.dx_stride, a.width, 4);
  dx.sums = p.dx_sums ? (float *)(ws + p.dx) : nullptr;
  dx.sums_ld = (uint64_t)ntiles * p.nt;
  dx.sums_split = a.tokens * dx.sums_ld;
  for (uint64_t k = 0; k < p.pieces; ++k) {
    const uint64_t row0 = k * p.piece, rows = std::min(p.piece, a.rows - row0);
    LogitDev l = logits(a, row0, rows);
    l.dloss = g.d_dloss;
    l.d = ws + p.d;
    l.d_ld = p.piece;
    const uint32_t grid = xcd_grid((uint64_t)l.ttiles * l.sweeps);
    if (direct)
      k_loss_d<DirectLogits, bf16><<<grid, 256, 0, st>>>(l);
    else if (a.dtype == NSFPS_F32)
      k_loss_d<StagedLogits<float, 3>, float><<<grid, 256, 0, st>>>(l);
    else if (one)
      k_loss_d<StagedLogits<bf16, 1>, bf16><<<grid, 256, 0, st>>>(l);
    else
      k_loss_d<StagedLogits<bf16, 1>, float><<<grid, 256, 0, st>>>(l);
    LAUNCH(hipGetLastError());

    const Matrix d = {ws + p.d, p.piece, (uint32_t)(direct ? p.tokens : a.tokens), (uint32_t)rows};
    dx.m = d;
    dx.n = l.e;
    dx.terms = (uint32_t)rows;
    dx.splits = p.dx_splits;  // those of a short last piece may be empty: they add nothing
    dx.add = k > 0;
    ProductDev de = dx;
    de.n = direct ? Matrix{ws + p.x, a.width, (uint32_t)p.tokens, a.width} : x;
    de.targets = direct ? nullptr : a.d_targets;
    de.vocabulary = (uint32_t)a.rows;
    de.mtiles = (uint32_t)host_ceil_div(rows, kTile);
    de.terms = (uint32_t)a.tokens;
    de.splits = p.de_splits;
    de.out = (char *)g.d_dtable + row0 * g.dtable_stride * z;
    de.out_ld = g.dtable_stride;
    de.out_rows = (uint32_t)rows;
    de.out_dtype = g.grad_dtype;
    de.out_wide = wide_any(g.grad_dtype, de.out, de.out_ld, a.width, 4);
    de.sums = p.de_sums ? (float *)(ws + p.de) : nullptr;
    de.sums_split = p.piece * de.sums_ld;
    de.add = 0;
    const uint32_t work = xcd_grid((uint64_t)dx.mtiles * ntiles * dx.splits +
                                   (uint64_t)de.mtiles * ntiles * de.splits);
    const auto products = [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      if (direct)
        k_loss_products_direct<NT><<<work, 256, 0, st>>>(dx, de);
      else if (a.dtype == NSFPS_F32)
        k_loss_products<float, 3, 3, float, 3, NT><<<work, 256, 0, st>>>(dx, de);
      else if (one)
        k_loss_products<bf16, 1, 1, bf16, 1, NT><<<work, 256, 0, st>>>(dx, de);
      else
        k_loss_products<float, 1, 2, bf16, 1, NT><<<work, 256, 0, st>>>(dx, de);
      return hipGetLastError();
    };
    LAUNCH(p.nt == 64 ? products(std::integral_constant<int, 2>())
                      : products(std::integral_constant<int, 4>()));
    if (de.sums) LAUNCH(write_out(de, st));
  }
  return dx.sums ? write_out(dx, st) : hipSuccess;
}

hipError_t preload_loss_kernels() {
  return func_attributes(k_loss_stats<DirectLogits>, k_loss_join<bf16>, k_loss_d<DirectLogits, bf16>,
                         k_loss_products_direct<4>, k_loss_out<bf16, 8>, k_loss_rows);
}

}  // namespace nsfps
