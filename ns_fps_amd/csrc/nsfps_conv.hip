// Short causal convolution with SiLU, its ring cache, and its gradient.
//
// y[t] = silu(bias + sum_k weight[k] x[t - (W-1) + k]) per channel.  A thread
// keeps a vector of channels and walks a tile of tokens with the last W inputs
// in registers, so each input row is read once (and W - 1 rows more per tile,
// from the caches).  Memory is the bound.
//
// Gradient, with pre the sum and sig its sigmoid:
//   g[t] = dy[t] sig (1 + pre (1 - sig)),  dx[t] = sum_k weight[k] g[t + W-1 - k],
//   dweight[k] = sum_t g[t] x[t - (W-1) + k],  dbias = sum_t g[t].
// The same walk finds pre again from x, so nothing is kept from the forward
// pass; g runs W - 1 tokens past the tile.  Parameter sums stay in registers
// over the tile, are added in a workgroup through LDS, and a second kernel
// adds the workgroups' sums in order.
//
// Measured, of 4.8 TB/s that a large copy reaches: 16,384 tokens of 323 float32
// channels 10.8 us (3.9 TB/s); 64 ragged sequences of up to 4,096 tokens, 640
// bfloat16 channels, 141 us (4.1 TB/s), their gradient 276 us (3.1 TB/s) and
// the join of its sums 20 us.
#include "nsfps_launch.h"
#include "nsfps_seq_device.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

constexpr uint32_t kTile = 32;      // tokens of a thread's walk (>= W - 1: only tile 0 reads history)
constexpr uint32_t kGradTile = 32;  // the same of the gradient's
constexpr uint32_t kAhead = 4;      // rows loaded together
constexpr int kVec = 8;      // bfloat16 channels of a thread
constexpr int kGradVec = 8;  // the same of the gradient's (4: as fast, but twice the sums to join)

// A launch's sequences, as the kernels see them.
struct Seqs {
  uint64_t batch, length;
  const int32_t *lengths, *positions, *slots;
};

__device__ __forceinline__ uint32_t seq_length(const Seqs &s, uint32_t b) {
  if (!s.lengths) return (uint32_t)s.length;
  const int32_t n = s.lengths[b];
  return n < 0 ? 0u : min((uint32_t)n, (uint32_t)s.length);
}

template <typename T, int V, int W>
__device__ __forceinline__ void load_weights(const T *__restrict__ weight, uint32_t c,
                                             float (&w)[V * W]) {
  if constexpr (V == 1) {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      float t[1];
      load_f32<T, 1>(weight + (uint64_t)c * W + k, t);
      w[k] = t[0];
    }
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      float t[V];
      load_f32<T, V>(weight + ((uint64_t)c * W + k) * V, t);
#pragma unroll
      for (int j = 0; j < V; ++j) w[k * V + j] = t[j];
    }
  }
}

// A workgroup holds cvb channel vectors of `per` tiles of tokens, in its first
// cvb * per threads.
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void k_conv(nsfps_rows x, nsfps_rows y, Seqs s,
                                              const T *__restrict__ weight,
                                              const T *__restrict__ bias, T *cache, uint32_t vecs,
                                              uint32_t cvb, uint32_t per, uint32_t tiles, uint64_t work) {
  const uint32_t cgroups = ceil_div(vecs, cvb);
  const uint32_t cl = threadIdx.x % cvb, tl = threadIdx.x / cvb;
  const uint32_t tgroups = ceil_div(tiles, per);
  for (uint64_t i = blockIdx.x; i < work; i += gridDim.x) {
    // neighbouring workgroups: the same tokens, further channels
    const uint32_t c = (uint32_t)(i % cgroups) * cvb + cl;
    const uint64_t r = i / cgroups;
    const uint32_t tile = (uint32_t)(r % tgroups) * per + tl;
    const uint32_t b = (uint32_t)(r / tgroups);
    if (c >= vecs || tl >= per || tile >= tiles) continue;
    const uint32_t len = seq_length(s, b), t0 = tile * kTile;
    const T *xr = (const T *)x.p + (uint64_t)b * x.batch_stride + (uint64_t)c * V;
    T *yr = (T *)y.p + (uint64_t)b * y.batch_stride + (uint64_t)c * V;
    float w[V * W], bs[V] = {};
    load_weights<T, V, W>(weight, c, w);
    if (bias) load_f32<T, V>(bias + (uint64_t)c * V, bs);

    const int32_t slot = cache ? (s.slots ? s.slots[b] : (int32_t)b) : -1;
    const uint32_t pos = slot >= 0 && s.positions && s.positions[b] > 0 ? s.positions[b] : 0u;
    const uint64_t ring_row = (uint64_t)vecs * V;
    T *const ring = cache + (slot >= 0 ? (uint64_t)slot * W * ring_row : 0) + (uint64_t)c * V;

    float win[W][V];  // x[t - (W-1)] .. x[t]
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      const int64_t t = (int64_t)t0 - (W - 1) + k;
#pragma unroll
      for (int j = 0; j < V; ++j) win[k][j] = 0.f;
      if (t >= 0) {
        if (t < len) load_f32<T, V>(xr + t * x.row_stride, win[k]);
      } else if ((int64_t)pos + t >= 0 && pos) {
        load_f32<T, V>(ring + (uint64_t)((pos + t) % W) * ring_row, win[k]);
      }
    }
    // kFull: the whole tile lies inside the sequence
    const auto walk = [&](auto full) {
      constexpr bool kFull = decltype(full)::value;
      Raw<T, V> in[kAhead], next[kAhead];
      const auto load = [&](uint32_t t, Raw<T, V>(&o)[kAhead]) {
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
          o[a] = zero_raw<T, V>();
          if (kFull || t + a < len) o[a] = load_raw<T, V>(xr + (uint64_t)(t + a) * x.row_stride);
        }
      };
      load(t0, in);
#pragma unroll 1
      for (uint32_t i = 0; i < kTile; i += kAhead) {
        if (i + kAhead < kTile) load(t0 + i + kAhead, next);
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
          const uint32_t t = t0 + i + a;
          numbers<T, V>(in[a], win[W - 1]);
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float pre = bs[j];
#pragma unroll
            for (int k = 0; k < W; ++k) pre = fmaf(w[j * W + k], win[k][j], pre);
            const float sig = sizeof(T) == 4 ? sigmoid(pre) : sigmoid_8bit(pre);
            o[j] = kFull || t < len ? pre * sig : 0.f;
          }
          if (kFull || t < s.length) store_f32<T, V>(yr + (uint64_t)t * y.row_stride, o);
#pragma unroll
          for (int k = 0; k < W - 1; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) win[k][j] = win[k + 1][j];
        }
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) in[a] = next[a];
      }
    };
    if ((uint64_t)t0 + kTile <= len)
      walk(std::true_type());
    else
      walk(std::false_type());
    // The thread that read the ring's history writes its new entries.
    if (tile == 0 && slot >= 0) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const int64_t t = (int64_t)len - W + k;
        if (t < 0) continue;
        float v[V];
        load_f32<T, V>(xr + t * x.row_stride, v);
        store_f32<T, V>(ring + (uint64_t)((pos + t) % W) * ring_row, v);
      }
    }
  }
}

// part: per workgroup of (sequence, tiles), per channel: W weight sums, one bias sum
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void k_conv_grad(nsfps_rows x, nsfps_rows dy, nsfps_rows dx,
                                                   Seqs s, const T *__restrict__ weight,
                                                   const T *__restrict__ bias,
                                                   float *__restrict__ part, uint32_t vecs,
                                                   uint32_t cvb, uint32_t per, uint32_t tiles, uint64_t work) {
  constexpr int kSums = V * (W + 1);
  __shared__ float s_sum[kSums][256];
  const uint32_t cgroups = ceil_div(vecs, cvb);
  const uint32_t cl = threadIdx.x % cvb, tl = threadIdx.x / cvb;
  const uint32_t tgroups = ceil_div(tiles, per);
  for (uint64_t i = blockIdx.x; i < work; i += gridDim.x) {
    const uint32_t c = (uint32_t)(i % cgroups) * cvb + cl;
    const uint64_t r = i / cgroups;
    const uint32_t tile = (uint32_t)(r % tgroups) * per + tl;
    const uint32_t b = (uint32_t)(r / tgroups);
    const bool mine = c < vecs && tl < per && tile < tiles;
    float dw[V][W] = {}, db[V] = {};
    if (mine) {
      const uint32_t len = seq_length(s, b), t0 = tile * kGradTile;
      const T *xr = (const T *)x.p + (uint64_t)b * x.batch_stride + (uint64_t)c * V;
      const T *gr = (const T *)dy.p + (uint64_t)b * dy.batch_stride + (uint64_t)c * V;
      T *dr = (T *)dx.p + (uint64_t)b * dx.batch_stride + (uint64_t)c * V;
      float w[V * W], bs[V] = {};
      load_weights<T, V, W>(weight, c, w);
      if (bias) load_f32<T, V>(bias + (uint64_t)c * V, bs);
      float win[W][V], g[W][V] = {};  // g[k] = g[t - k]
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        const int64_t t = (int64_t)t0 - (W - 1) + k;
#pragma unroll
        for (int j = 0; j < V; ++j) win[k][j] = 0.f;
        if (t >= 0 && t < len) load_f32<T, V>(xr + t * x.row_stride, win[k]);
      }
      // kFull: the tile and the W - 1 tokens after it lie inside the sequence
      constexpr uint32_t kSteps = (kGradTile + W - 1 + kAhead - 1) / kAhead * kAhead;
      const auto walk = [&](auto full) {
        constexpr bool kFull = decltype(full)::value;
        Raw<T, V> in[kAhead], gi[kAhead], next[kAhead], gnext[kAhead];
        const auto load = [&](uint32_t t, Raw<T, V>(&o)[kAhead], Raw<T, V>(&go)[kAhead]) {
#pragma unroll
          for (uint32_t a = 0; a < kAhead; ++a) {
            o[a] = go[a] = zero_raw<T, V>();
            if (kFull || t + a < len) {
              o[a] = load_raw<T, V>(xr + (uint64_t)(t + a) * x.row_stride);
              go[a] = load_raw<T, V>(gr + (uint64_t)(t + a) * dy.row_stride);
            }
          }
        };
        load(t0, in, gi);
#pragma unroll 1
        for (uint32_t i = 0; i < kSteps; i += kAhead) {
          if (i + kAhead < kSteps) load(t0 + i + kAhead, next, gnext);
#pragma unroll
          for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t t = t0 + i + a;
            const bool counts = i + a < kGradTile;  // the tile's own tokens
            float gv[V];
            numbers<T, V>(in[a], win[W - 1]);
            numbers<T, V>(gi[a], gv);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              float pre = bs[j];
#pragma unroll
              for (int k = 0; k < W; ++k) pre = fmaf(w[j * W + k], win[k][j], pre);
              const Logistic s1 = logistic(pre);
              // past the sequence's end the slope counts for nothing, not even as NaN
              const float gt = kFull || t < len ? gv[j] * s1.sig * fmaf(pre, s1.rest, 1.f) : 0.f;
#pragma unroll
              for (int k = W - 1; k > 0; --k) g[k][j] = g[k - 1][j];
              g[0][j] = gt;
              if (counts) {
                db[j] += gt;
#pragma unroll
                for (int k = 0; k < W; ++k) dw[j][k] = fmaf(gt, win[k][j], dw[j][k]);
              }
#pragma unroll
              for (int k = 0; k < W - 1; ++k) win[k][j] = win[k + 1][j];
            }
            if (i + a >= W - 1 && i + a < kGradTile + W - 1) {  // g[t - (W-1) .. t] are known
              const uint32_t to = t - (W - 1);
              float o[V];
#pragma unroll
              for (int j = 0; j < V; ++j) {
                o[j] = 0.f;
#pragma unroll
                for (int k = 0; k < W; ++k) o[j] = fmaf(w[j * W + k], g[k][j], o[j]);
              }
              if (kFull || to < s.length) store_f32<T, V>(dr + (uint64_t)to * dx.row_stride, o);
            }
          }
#pragma unroll
          for (uint32_t a = 0; a < kAhead; ++a) in[a] = next[a], gi[a] = gnext[a];
        }
      };
      if ((uint64_t)t0 + kSteps <= len)
        walk(std::true_type());
      else
        walk(std::false_type());
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int k = 0; k < W; ++k) s_sum[j * (W + 1) + k][threadIdx.x] = dw[j][k];
      s_sum[j * (W + 1) + W][threadIdx.x] = db[j];
    }
    __syncthreads();
    // sums of a channel vector: kSums floats next to each other in part
    for (uint32_t e = threadIdx.x; e < cvb * kSums; e += blockDim.x) {
      const uint32_t lc = e / kSums, k = e % kSums;
      const uint32_t cc = (uint32_t)(i % cgroups) * cvb + lc;
      if (cc >= vecs) continue;
      float t = 0.f;
      for (uint32_t p = 0; p < per; ++p) t += s_sum[k][p * cvb + lc];
      part[r * ((uint64_t)vecs * kSums) + (uint64_t)cc * kSums + k] = t;
    }
    __syncthreads();
  }
}

// out[e] = the sum over rows of part[row][e], e a channel's weight or bias sum
__global__ __launch_bounds__(1024) void k_conv_join(const float *__restrict__ part, uint64_t rows,
                                                    uint64_t cols, uint32_t w1,
                                                    float *__restrict__ dweight,
                                                    float *__restrict__ dbias) {
  __shared__ float s_sum[16][64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint64_t e = (uint64_t)blockIdx.x * 64 + lane;
  const uint64_t run = (rows + 15) / 16;
  const uint64_t a = min(wave * run, rows), z = min(a + run, rows);
  float acc = 0.f;
  if (e < cols) {
    uint64_t r = a;
    for (; r + 8 <= z; r += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(r + k) * cols + e];
#pragma unroll
      for (int k = 0; k < 8; ++k) acc += v[k];
    }
    for (; r < z; ++r) acc += part[r * cols + e];
  }
  s_sum[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && e < cols) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += s_sum[w][lane];
    const uint64_t c = e / w1;
    const uint32_t k = (uint32_t)(e % w1);
    if (k + 1 < w1)
      dweight[c * (w1 - 1) + k] = t;
    else if (dbias)
      dbias[c] = t;
  }
}

struct Shape {
  uint32_t vecs, cvb, per, threads, tiles;
  uint64_t rows, work;  // (sequence, tile group) pairs; times channel groups
};

// All channel vectors in one workgroup where 256 threads hold them, else equal
// parts of them; then as many tiles of tokens as fit.
Shape shape_of(const nsfps_conv_args &a, uint32_t v, uint32_t tile) {
  Shape s;
  s.vecs = a.channels / v;
  s.cvb = (uint32_t)host_ceil_div(s.vecs, host_ceil_div(s.vecs, 256));
  s.tiles = (uint32_t)host_ceil_div(a.length, tile);
  s.per = std::max(1u, std::min(256 / s.cvb, s.tiles));
  s.threads = (s.cvb * s.per + 63) & ~63u;
  s.rows = a.batch * host_ceil_div(s.tiles, s.per);
  s.work = s.rows * host_ceil_div(s.vecs, s.cvb);
  return s;
}

Seqs seqs_of(const nsfps_conv_args &a) {
  return Seqs{a.batch, a.length, a.d_lengths, a.d_positions, a.d_slots};
}

uint32_t grid_of(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, 1u << 20); }

// f(element type, elements a vector, width)
template <int kBf16, typename F>
hipError_t by_type(uint32_t dtype, bool wide, uint32_t width, F f) {
  const auto by_width = [&](auto t, auto v) {
    switch (width) {
      case 2: return f(t, v, std::integral_constant<int, 2>());
      case 3: return f(t, v, std::integral_constant<int, 3>());
      default: return f(t, v, std::integral_constant<int, 4>());
    }
  };
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 4> four;
  constexpr std::integral_constant<int, kBf16> many;
  if (dtype == NSFPS_F32) return wide ? by_width(float(), four) : by_width(float(), one);
  return wide ? by_width(bf16(), many) : by_width(bf16(), one);
}

// Vectors of a lane fit the channels, the parameters and the rows.
bool conv_wide(const nsfps_conv_args &a, uint32_t bf16s, std::initializer_list<const nsfps_rows *> rows) {
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2, v = a.dtype == NSFPS_F32 ? 4 : bf16s;
  const auto at = [&](const void *p) { return (uintptr_t)p % (v * size) == 0; };
  bool ok = a.channels % v == 0 && at(a.d_weight) && at(a.d_bias) && at(a.d_cache);
  for (const nsfps_rows *r : rows)
    ok = ok && at(r->p) && r->batch_stride % v == 0 && r->row_stride % v == 0;
  return ok;
}

}  // namespace

hipError_t launch_conv(const nsfps_conv_args &a, hipStream_t st) {
  const bool wide = conv_wide(a, kVec, {&a.x, &a.y});
  return by_type<kVec>(a.dtype, wide, a.width, [&](auto t, auto v, auto w) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, W = decltype(w)::value;
    const Shape s = shape_of(a, V, kTile);
    k_conv<T, V, W><<<grid_of(s.work), s.threads, 0, st>>>(
        a.x, a.y, seqs_of(a), (const T *)a.d_weight, (const T *)a.d_bias, (T *)a.d_cache, s.vecs,
        s.cvb, s.per, s.tiles, s.work);
    return hipGetLastError();
  });
}

uint64_t conv_grad_bytes(const nsfps_conv_args &a) {
  // what the strides allow is not known here: the most of the forms
  uint64_t rows = 0;
  for (uint32_t v : {1u, 4u, (uint32_t)kGradVec})
    if (a.channels % v == 0) rows = std::max(rows, shape_of(a, v, kGradTile).rows);
  return rows * a.channels * (a.width + 1) * 4;
}

hipError_t launch_conv_grad(const nsfps_conv_args &a, const nsfps_conv_grads &g, hipStream_t st) {
  const bool wide = conv_wide(a, kGradVec, {&a.x, &g.dy, &g.dx});
  return by_type<kGradVec>(a.dtype, wide, a.width, [&](auto t, auto v, auto w) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value, W = decltype(w)::value;
    const Shape s = shape_of(a, V, kGradTile);
    float *const part = (float *)a.workspace;
    if (s.work)
      k_conv_grad<T, V, W><<<grid_of(s.work), s.threads, 0, st>>>(
          a.x, g.dy, g.dx, seqs_of(a), (const T *)a.d_weight, (const T *)a.d_bias, part, s.vecs,
          s.cvb, s.per, s.tiles, s.work);
    const uint64_t cols = (uint64_t)a.channels * (W + 1);
    k_conv_join<<<(uint32_t)host_ceil_div(cols, 64), 1024, 0, st>>>(part, s.rows, cols, W + 1,
                                                                   g.d_dweight, g.d_dbias);
    return hipGetLastError();
  });
}

hipError_t preload_conv_kernels() {
  return func_attributes(k_conv<bf16, kVec, 4>, k_conv_grad<bf16, kGradVec, 4>, k_conv_join);
}

}  // namespace nsfps
