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
// Operands of the products are bfloat16.  A float32 value enters as three
// bfloat16 terms whose sum it is, in planes behind each other, and a product
// of float32 values as the six products of terms that reach 24 bits.  d is
// rounded to one term (8 bits) where the products' results are bfloat16, to two
// for a float32 table gradient of bfloat16 inputs, to three in float32 calls.
// Sums are float32 everywhere.
#include "nsfps_launch.h"
#include "nsfps_product.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

constexpr uint32_t kTile = 128;  // tokens and vocabulary rows of a tile

// The products of planes that make one product: plane of m, plane of n, two
// bits each, the smallest first.
struct Passes {
  uint32_t n, m_code, n_code;
};
constexpr Passes kPassesOne = {1, 0, 0};
// (1, 0), (0, 0): two terms of m, one of n
constexpr Passes kPassesTwo = {2, 1, 0};
// (2, 0) (0, 2) (1, 1) (1, 0) (0, 1) (0, 0)
constexpr Passes kPassesSix = {6, 2 | 0 << 2 | 1 << 4 | 1 << 6, 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8};

struct Operand {
  const bf16 *p;
  uint64_t ld, plane;  // elements from row to row, from plane to plane
};

// ---- packing: rows of bfloat16 terms, padded with zeros

// planes of [out_rows][out_width]; a row whose target is outside the vocabulary
// is zeros too (targets null: none is)
template <typename T, int P>
__global__ __launch_bounds__(256) void k_loss_pack(const T *__restrict__ in, uint64_t stride,
                                                   uint32_t rows, uint32_t width,
                                                   const int32_t *__restrict__ targets,
                                                   uint32_t vocabulary, bf16 *__restrict__ out,
                                                   uint64_t out_rows, uint32_t out_width) {
  const uint32_t vecs = out_width / 8;
  const uint64_t work = out_rows * vecs;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < work;
       i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = i / vecs;
    const uint32_t c = (uint32_t)(i % vecs) * 8;
    float v[8];
    const bool row = r < rows && (!targets || (uint32_t)targets[r] < vocabulary);
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      v[k] = 0.f;
      if (row && c + k < width) load_f32<T, 1>(in + r * stride + c + k, *(float(*)[1])&v[k]);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      store_f32<bf16, 8>(out + (p * out_rows + r) * out_width + c, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] -= to_f32(bf16{bf16_bits(v[k])});
    }
  }
}

// ---- tiles of z

struct LogitDev {
  Operand x, e;
  Passes passes;
  uint32_t ksteps;            // stages of one pass
  uint32_t tokens, rows;      // rows: of the piece
  uint32_t ttiles, vtiles;    // tiles of tokens, of the piece's vocabulary
  uint32_t sweep, sweeps;     // vocabulary tiles a workgroup takes one after another
  float scale2;               // scale * log2(e)
  // statistics
  float2 *parts;              // [parts][tokens padded]: maximum and sum, in powers of two
  uint32_t part0;             // of the piece
  uint64_t part_stride;
  // gradient
  const float *lse, *dloss;
  const int32_t *targets;
  uint32_t row0, vocabulary;  // the piece's first row, rows of the whole table
  float scale;
  bf16 *d;                    // planes of [tokens padded][d_ld]
  uint64_t d_ld, d_plane;
};

typedef Product<2, 2, 4, 4, false, false, true> LogitProduct;

// Walks the sweep of a workgroup; epilogue(sum, vocabulary tile) for each tile.
template <typename F>
__device__ __forceinline__ void logit_tiles(const LogitDev &a, LogitProduct::Lds &lds,
                                            uint32_t ttile, uint32_t first, uint32_t last,
                                            F epilogue) {
  LogitProduct product;
  product.fm.start(a.x.p + (uint64_t)ttile * kTile * a.x.ld, a.x.ld);
  product.fn.start(a.e.p + (uint64_t)first * kTile * a.e.ld, a.e.ld);
  const uint32_t steps = a.passes.n * a.ksteps;
  // the stage issued next: tile, pass, step
  uint32_t tile = first, pass = 0, k = 0, buf = 0;
  const auto issue = [&](uint32_t b) {
    const uint64_t mp = a.passes.m_code >> (2 * pass) & 3, np = a.passes.n_code >> (2 * pass) & 3;
    product.issue(lds, b, mp * a.x.plane + k * kStage,
                  np * a.e.plane + (uint64_t)(tile - first) * kTile * a.e.ld + k * kStage);
    if (++k == a.ksteps) {
      k = 0;
      if (++pass == a.passes.n) pass = 0, ++tile;
    }
  };
  issue(0);
  for (uint32_t t = first; t < last; ++t) {
    f32x4 sum[4][4] = {};
    for (uint32_t s = 0; s < steps; ++s) {
      product.add(sum, lds, buf, [&] {
        if (tile < last) issue(buf ^ 1);
      });
      buf ^= 1;
    }
    epilogue(sum, t);
  }
}

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

__device__ __forceinline__ void join_stats(float &m, float &s, float m2, float s2) {
  const float top = fmaxf(m, m2), at = top == -INFINITY ? 0.f : top;
  s = s * exp2_fast(m - at) + s2 * exp2_fast(m2 - at);
  m = top;
}

__global__ __launch_bounds__(256, 2) void k_loss_stats(LogitDev a) {
  __shared__ LogitProduct::Lds lds;
  uint32_t ttile, first, last;
  if (!logit_item(a, ttile, first, last)) return;
  const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / 2, wn = wave % 2;
  float top[4], sum[4];  // of this lane's columns, for its four tokens
#pragma unroll
  for (int i = 0; i < 4; ++i) top[i] = -INFINITY, sum[i] = 0.f;
  logit_tiles(a, lds, ttile, first, last, [&](f32x4(&z)[4][4], uint32_t tile) {
    const uint32_t v0 = tile * kTile + 64 * wn + 16 * g;
    const bool ragged = (tile + 1) * kTile > a.rows;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float m = top[i];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v = z[i][j][r] * a.scale2;
          if (ragged && v0 + 4 * j + r >= a.rows) v = -INFINITY;
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
    const uint32_t token = ttile * kTile + 64 * wm + 16 * i + l;
    if (g == 0)
      a.parts[(uint64_t)(a.part0 + first / a.sweep * 2 + wn) * a.part_stride + token] =
          make_float2(top[i], sum[i]);
  }
}

// lse and loss: a wave a token joins the parts and finds the target's logit.
template <typename T>
__global__ __launch_bounds__(256) void k_loss_join(const float2 *__restrict__ parts, uint32_t nparts,
                                                   uint64_t part_stride, uint32_t tokens,
                                                   const T *__restrict__ x, uint64_t x_stride,
                                                   const T *__restrict__ table,
                                                   uint64_t table_stride, uint32_t rows,
                                                   uint32_t width, float scale,
                                                   const int32_t *__restrict__ targets,
                                                   float *__restrict__ loss,
                                                   float *__restrict__ lse) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint64_t i = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < tokens;
       i += (uint64_t)gridDim.x * 4) {
    const uint32_t target = (uint32_t)targets[i];
    float dot = 0.f;
    if (target < rows) {
      const T *xr = x + i * x_stride, *er = table + (uint64_t)target * table_stride;
      for (uint32_t c = lane; c < width; c += 64) {
        float u[1], v[1];
        load_f32<T, 1>(xr + c, u);
        load_f32<T, 1>(er + c, v);
        dot = fmaf(u[0], v[0], dot);
      }
    }
    float m = -INFINITY, s = 0.f;
    for (uint32_t p = lane; p < nparts; p += 64) {
      const float2 v = parts[p * part_stride + i];
      join_stats(m, s, v.x, v.y);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      dot += __shfl_xor(dot, off, 64);
      join_stats(m, s, __shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
    }
    if (lane == 0) {
      const float all = (m + log2f(s)) * kLn2;
      lse[i] = all;
      loss[i] = target < rows ? all - scale * dot : 0.f;
    }
  }
}

// A piece's d.
template <int P>
__global__ __launch_bounds__(256, 2) void k_loss_d(LogitDev a) {
  __shared__ LogitProduct::Lds lds;
  uint32_t ttile, first, last;
  if (!logit_item(a, ttile, first, last)) return;
  const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / 2, wn = wave % 2;
  float lse2[4], weight[4];
  uint32_t target[4];  // in the piece
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t token = ttile * kTile + 64 * wm + 16 * i + l;
    lse2[i] = weight[i] = 0.f;
    target[i] = ~0u;
    if (token < a.tokens && (uint32_t)a.targets[token] < a.vocabulary) {
      lse2[i] = a.lse[token] * kLog2e;
      weight[i] = a.dloss[token] * a.scale;
      target[i] = (uint32_t)a.targets[token] - a.row0;
    }
  }
  logit_tiles(a, lds, ttile, first, last, [&](f32x4(&z)[4][4], uint32_t tile) {
    const uint32_t v0 = tile * kTile + 64 * wn + 16 * g;
    const bool ragged = (tile + 1) * kTile > a.rows;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t token = ttile * kTile + 64 * wm + 16 * i + l, hit = target[i] - v0;
      float d[16];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p = exp2_fast(fmaf(z[i][j][r], a.scale2, -lse2[i]));
          if (hit == 4 * j + r) p -= 1.f;
          d[4 * j + r] = ragged && v0 + 4 * j + r >= a.rows ? 0.f : p * weight[i];
        }
      bf16 *const out = a.d + (uint64_t)token * a.d_ld + v0;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float lo[8], hi[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) lo[k] = d[k], hi[k] = d[8 + k];
        store_f32<bf16, 8>(out + p * a.d_plane, lo);
        store_f32<bf16, 8>(out + p * a.d_plane + 8, hi);
#pragma unroll
        for (int k = 0; k < 16; ++k) d[k] -= to_f32(bf16{bf16_bits(d[k])});
      }
    }
  });
}

// ---- the products of d

struct ProductDev {
  Operand m, n;
  Passes passes;
  uint32_t mtiles, ntiles;
  uint32_t ksteps, per, splits;  // stages of one pass, of a split, splits
  float *c;                      // [splits][rows of m][ldc]
  uint64_t c_split, ldc;
  uint32_t add;                  // to what c holds
};

// dx: m = d by rows; dE: m = d by columns.  The other operand by columns.
template <bool kMCol, int NT>
__global__ __launch_bounds__(256, 2) void k_loss_product(ProductDev a) {
  typedef Product<2, 2, 4, NT, kMCol, true, false> P;
  __shared__ typename P::Lds lds;
  const uint32_t work = a.mtiles * a.ntiles * a.splits, per = (work + 7) / 8;
  const uint32_t w = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || w >= work) return;
  const uint32_t nt = w % a.ntiles, mt = w / a.ntiles % a.mtiles, split = w / a.ntiles / a.mtiles;
  const uint32_t k0 = split * a.per, k1 = min(k0 + a.per, a.ksteps);
  P product;
  const uint64_t m_step = kMCol ? kStage * a.m.ld : kStage, n_step = kStage * a.n.ld;
  product.fm.start(a.m.p + (kMCol ? (uint64_t)mt * P::kM : (uint64_t)mt * P::kM * a.m.ld), a.m.ld);
  product.fn.start(a.n.p + (uint64_t)nt * P::kN, a.n.ld);
  uint32_t pass = 0, k = k0, buf = 0;
  const auto issue = [&](uint32_t b) {
    const uint64_t mp = a.passes.m_code >> (2 * pass) & 3, np = a.passes.n_code >> (2 * pass) & 3;
    product.issue(lds, b, mp * a.m.plane + k * m_step, np * a.n.plane + k * n_step);
    if (++k == k1) k = k0, ++pass;
  };
  f32x4 sum[4][NT] = {};
  issue(0);
  const uint32_t steps = a.passes.n * (k1 - k0);
  for (uint32_t s = 0; s < steps; ++s) {
    product.add(sum, lds, buf, [&] {
      if (pass < a.passes.n) issue(buf ^ 1);
    });
    buf ^= 1;
  }
  const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, l = lane & 15u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / 2, wn = wave % 2;
  float *const c = a.c + split * a.c_split + ((uint64_t)mt * P::kM + 64 * wm + l) * a.ldc +
                   nt * P::kN + 16 * NT * wn + 4 * g;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      NSFPS_GLOBAL_SEQ f32x4 *at = (NSFPS_GLOBAL_SEQ f32x4 *)(c + 16 * i * a.ldc + 16 * j);
      *at = a.add ? *at + sum[i][j] : sum[i][j];
    }
}

// The splits' sums, added in order, as rows of the result.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_loss_out(const float *__restrict__ c, uint64_t c_split,
                                                  uint64_t ldc, uint32_t splits, T *__restrict__ out,
                                                  uint64_t stride, uint64_t rows, uint32_t width) {
  const uint32_t vecs = (width + V - 1) / V;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < rows * vecs;
       i += (uint64_t)gridDim.x * 256) {
    const uint64_t r = i / vecs, at = r * ldc + (i % vecs) * V;
    float v[V] = {};
    for (uint32_t s = 0; s < splits; ++s) {
      float t[V];
      constexpr int W = V < 4 ? V : 4;
#pragma unroll
      for (int k = 0; k < V; k += W) load_f32<float, W>(c + s * c_split + at + k, *(float(*)[W])&t[k]);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] += t[k];
    }
    store_f32<T, V>(out + r * stride + (i % vecs) * V, v);
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

struct Plan {
  uint32_t planes, width;      // planes of an input; columns of packed rows
  uint64_t tokens;             // padded
  uint64_t piece;              // vocabulary rows of a piece, a multiple of kTile
  uint64_t pieces;
  uint32_t d_planes, nt;       // gradient: planes of d; columns of a product's tile
  uint32_t dx_splits, de_splits, dx_per, de_per;
  uint32_t ttiles, vtiles, sweep, sweeps;  // of a whole piece
  uint64_t x, e, parts, d, dx, de, bytes;  // workspace offsets
};

void plan_splits(uint64_t tiles, uint64_t ksteps, uint32_t &per, uint32_t &splits) {
  constexpr uint64_t kFill = 512, kLeast = 4;
  const uint64_t want = std::max<uint64_t>(1, kFill / std::max<uint64_t>(1, tiles));
  per = (uint32_t)std::max<uint64_t>(std::min(kLeast, ksteps), host_ceil_div(ksteps, want));
  splits = (uint32_t)host_ceil_div(ksteps, per);
}

Plan plan_of(uint64_t tokens, uint64_t rows, uint32_t width, uint32_t dtype, bool grad,
             uint32_t grad_dtype) {
  Plan p = {};
  p.planes = dtype == NSFPS_F32 ? 3 : 1;
  p.width = (uint32_t)(width <= 64 ? 64 : up(width, 128));
  p.tokens = up(tokens, kTile);
  const uint64_t whole = up(rows, kTile);
  if (!p.tokens || !whole) {
    p.bytes = 256;
    return p;
  }
  // a piece of d: 64 million values, and 1,024 rows at least
  constexpr uint64_t kValues = 1ull << 26;
  p.piece = std::min(whole, std::max<uint64_t>(1024, kValues / p.tokens / kTile * kTile));
  p.pieces = host_ceil_div(whole, p.piece);
  p.ttiles = (uint32_t)(p.tokens / kTile);
  p.vtiles = (uint32_t)(p.piece / kTile);
  const uint64_t fill = std::max<uint64_t>(1, (uint64_t)p.ttiles * p.vtiles / 1024);
  p.sweep = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(p.vtiles, 16), fill);
  p.sweeps = (p.vtiles + p.sweep - 1) / p.sweep;
  uint64_t at = 0;
  const auto take = [&](uint64_t n) {
    const uint64_t was = at;
    at += bytes256(n);
    return was;
  };
  p.x = take(2 * p.planes * p.tokens * p.width);
  p.e = take(2 * p.planes * p.piece * p.width);
  if (!grad) {
    p.parts = take(8 * 2 * p.sweeps * p.pieces * p.tokens);
  } else {
    p.d_planes = dtype == NSFPS_F32 ? 3 : grad_dtype == NSFPS_F32 ? 2 : 1;
    p.nt = p.width == 64 ? 64 : 128;
    p.d = take(2 * p.d_planes * p.tokens * p.piece);
    plan_splits(p.ttiles * (uint64_t)(p.width / p.nt), p.piece / kStage, p.dx_per, p.dx_splits);
    plan_splits(p.vtiles * (uint64_t)(p.width / p.nt), p.tokens / kStage, p.de_per, p.de_splits);
    p.dx = take(4 * p.dx_splits * p.tokens * p.width);
    p.de = take(4 * p.de_splits * p.piece * p.width);
  }
  p.bytes = std::max<uint64_t>(256, at);
  return p;
}

struct Call {
  const nsfps_loss_args &a;
  const Plan &p;
  char *ws;
  hipStream_t st;

  template <typename T>
  hipError_t pack(const void *in, uint64_t stride, uint64_t rows, const int32_t *targets,
                  bf16 *out, uint64_t out_rows) const {
    k_loss_pack<T, sizeof(T) == 4 ? 3 : 1><<<grid_of(out_rows * p.width / 8), 256, 0, st>>>(
        (const T *)in, stride, (uint32_t)rows, a.width, targets, (uint32_t)a.rows, out, out_rows,
        p.width);
    return hipGetLastError();
  }
  hipError_t pack_any(const void *in, uint64_t stride, uint64_t rows, const int32_t *targets,
                      uint64_t at, uint64_t out_rows) const {
    bf16 *const out = (bf16 *)(ws + at);
    return a.dtype == NSFPS_F32 ? pack<float>(in, stride, rows, targets, out, out_rows)
                                : pack<bf16>(in, stride, rows, targets, out, out_rows);
  }
  uint64_t size() const { return a.dtype == NSFPS_F32 ? 4 : 2; }
  // rows of piece number k
  uint64_t piece_rows(uint64_t k) const { return std::min(p.piece, a.rows - k * p.piece); }
  hipError_t pack_piece(uint64_t k) const {
    return pack_any((const char *)a.d_table + k * p.piece * a.table_stride * size(), a.table_stride,
                    piece_rows(k), nullptr, p.e, p.piece);
  }
  Passes passes() const { return a.dtype == NSFPS_F32 ? kPassesSix : kPassesOne; }
  LogitDev logits(uint64_t k) const {
    LogitDev d = {};
    d.x = {(const bf16 *)(ws + p.x), p.width, p.tokens * p.width};
    d.e = {(const bf16 *)(ws + p.e), p.width, p.piece * p.width};
    d.passes = passes();
    d.ksteps = p.width / kStage;
    d.tokens = (uint32_t)a.tokens;
    d.rows = (uint32_t)piece_rows(k);
    d.ttiles = p.ttiles;
    d.vtiles = p.vtiles;
    d.sweep = p.sweep;
    d.sweeps = p.sweeps;
    d.scale = a.scale;
    d.scale2 = a.scale * kLog2e;
    d.parts = (float2 *)(ws + p.parts);
    d.part0 = (uint32_t)(2 * p.sweeps * k);
    d.part_stride = p.tokens;
    d.row0 = (uint32_t)(k * p.piece);
    d.vocabulary = (uint32_t)a.rows;
    d.targets = a.d_targets;
    d.lse = a.d_lse;
    d.d = (bf16 *)(ws + p.d);
    d.d_ld = p.piece;
    d.d_plane = p.tokens * p.piece;
    return d;
  }
};

uint32_t xcd_grid(uint64_t work) { return (uint32_t)((work + 7) / 8 * 8); }

template <bool kMCol>
hipError_t run_product(const ProductDev &d, uint32_t nt, hipStream_t st) {
  const uint32_t grid = xcd_grid((uint64_t)d.mtiles * d.ntiles * d.splits);
  if (nt == 64)
    k_loss_product<kMCol, 2><<<grid, 256, 0, st>>>(d);
  else
    k_loss_product<kMCol, 4><<<grid, 256, 0, st>>>(d);
  return hipGetLastError();
}

template <typename T>
hipError_t write_rows(const float *c, uint64_t c_split, uint64_t ldc, uint32_t splits, void *out,
                      uint64_t stride, uint64_t rows, uint32_t width, hipStream_t st) {
  constexpr int V = kWide<T>;
  if (width % V == 0 && stride % V == 0 && (uintptr_t)out % 16 == 0)
    k_loss_out<T, V><<<grid_of(rows * (width / V)), 256, 0, st>>>(c, c_split, ldc, splits, (T *)out,
                                                                   stride, rows, width);
  else
    k_loss_out<T, 1><<<grid_of(rows * width), 256, 0, st>>>(c, c_split, ldc, splits, (T *)out, stride,
                                                            rows, width);
  return hipGetLastError();
}
hipError_t write_any(uint32_t dtype, const float *c, uint64_t c_split, uint64_t ldc, uint32_t splits,
                     void *out, uint64_t stride, uint64_t rows, uint32_t width, hipStream_t st) {
  return dtype == NSFPS_F32
             ? write_rows<float>(c, c_split, ldc, splits, out, stride, rows, width, st)
             : write_rows<bf16>(c, c_split, ldc, splits, out, stride, rows, width, st);
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

uint64_t loss_bytes(const nsfps_loss_args &a) {
  return plan_of(a.tokens, a.rows, a.width, a.dtype, false, 0).bytes;
}

hipError_t launch_loss(const nsfps_loss_args &a, hipStream_t st) {
  const Plan p = plan_of(a.tokens, a.rows, a.width, a.dtype, false, 0);
  const Call c{a, p, (char *)a.workspace, st};
  if (p.pieces) LAUNCH(c.pack_any(a.d_x, a.x_stride, a.tokens, nullptr, p.x, p.tokens));
  for (uint64_t k = 0; k < p.pieces; ++k) {
    LAUNCH(c.pack_piece(k));
    k_loss_stats<<<xcd_grid((uint64_t)p.ttiles * p.sweeps), 256, 0, st>>>(c.logits(k));
    LAUNCH(hipGetLastError());
  }
  const auto join = [&](auto t) {
    using T = decltype(t);
    k_loss_join<T><<<grid_of(a.tokens * 64), 256, 0, st>>>(
        (const float2 *)((char *)a.workspace + p.parts), (uint32_t)(2 * p.sweeps * p.pieces),
        p.tokens, (uint32_t)a.tokens, (const T *)a.d_x, a.x_stride, (const T *)a.d_table,
        a.table_stride, (uint32_t)a.rows, a.width, a.scale, a.d_targets, a.d_loss, a.d_lse);
    return hipGetLastError();
  };
  return a.dtype == NSFPS_F32 ? join(float()) : join(bf16());
}

uint64_t loss_grad_bytes(const nsfps_loss_args &a, const nsfps_loss_grads &g) {
  return plan_of(a.tokens, a.rows, a.width, a.dtype, true, g.grad_dtype).bytes;
}

hipError_t launch_loss_grad(const nsfps_loss_args &a, const nsfps_loss_grads &g, hipStream_t st) {
  const Plan p = plan_of(a.tokens, a.rows, a.width, a.dtype, true, g.grad_dtype);
  if (!p.pieces) {
    LAUNCH(write_zeros(a.dtype, g.d_dx, g.dx_stride, a.tokens, a.width, st));
    return write_zeros(g.grad_dtype, g.d_dtable, g.dtable_stride, a.rows, a.width, st);
  }
  const Call c{a, p, (char *)a.workspace, st};
  char *const ws = c.ws;
  // a row that counts for nothing may hold anything: it enters as zeros
  LAUNCH(c.pack_any(a.d_x, a.x_stride, a.tokens, a.d_targets, p.x, p.tokens));
  const Operand x = {(const bf16 *)(ws + p.x), p.width, p.tokens * p.width},
                e = {(const bf16 *)(ws + p.e), p.width, p.piece * p.width},
                d = {(const bf16 *)(ws + p.d), p.piece, p.tokens * p.piece};
  float *const dx = (float *)(ws + p.dx), *const de = (float *)(ws + p.de);
  for (uint64_t k = 0; k < p.pieces; ++k) {
    LAUNCH(c.pack_piece(k));
    LogitDev l = c.logits(k);
    l.dloss = g.d_dloss;
    const uint32_t grid = xcd_grid((uint64_t)p.ttiles * p.sweeps);
    if (p.d_planes == 3)
      k_loss_d<3><<<grid, 256, 0, st>>>(l);
    else if (p.d_planes == 2)
      k_loss_d<2><<<grid, 256, 0, st>>>(l);
    else
      k_loss_d<1><<<grid, 256, 0, st>>>(l);
    LAUNCH(hipGetLastError());
    ProductDev q = {};
    q.m = d;
    q.n = e;
    q.passes = c.passes();
    q.mtiles = p.ttiles;
    q.ntiles = p.width / p.nt;
    q.ksteps = (uint32_t)(p.piece / kStage);
    q.per = p.dx_per;
    q.splits = p.dx_splits;
    q.c = dx;
    q.ldc = p.width;
    q.c_split = p.tokens * p.width;
    q.add = k > 0;
    LAUNCH(run_product<false>(q, p.nt, st));
    q.n = x;
    q.passes = p.d_planes == 3 ? kPassesSix : p.d_planes == 2 ? kPassesTwo : kPassesOne;
    q.mtiles = p.vtiles;
    q.ksteps = (uint32_t)(p.tokens / kStage);
    q.per = p.de_per;
    q.splits = p.de_splits;
    q.c = de;
    q.c_split = p.piece * p.width;
    q.add = 0;
    LAUNCH(run_product<true>(q, p.nt, st));
    const uint64_t z = g.grad_dtype == NSFPS_F32 ? 4 : 2;
    LAUNCH(write_any(g.grad_dtype, de, q.c_split, p.width, p.de_splits,
                     (char *)g.d_dtable + k * p.piece * g.dtable_stride * z, g.dtable_stride,
                     c.piece_rows(k), a.width, st));
  }
  return write_any(a.dtype, dx, p.tokens * p.width, p.width, p.dx_splits, g.d_dx, g.dx_stride,
                   a.tokens, a.width, st);
}

hipError_t preload_loss_kernels() {
  return func_attributes(k_loss_pack<bf16, 1>, k_loss_stats, k_loss_join<bf16>, k_loss_d<1>,
                         k_loss_product<false, 4>, k_loss_product<true, 4>, k_loss_out<bf16, 8>);
}

}  // namespace nsfps
