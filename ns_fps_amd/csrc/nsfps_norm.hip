// Norms of queries and keys by head with the rotation by their position, and
// their gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = r x,  y = R (w n)
// R turns the pair number i by position * freq[i].  With g = R^T dy:
//   dw = sum over tokens and heads of g n,  dx = r (g w - n mean(g w n)).
//
// A group of lanes holds a head's values as slots of two: a rotated pair, or
// two values behind the rotation (whose angle is 0), a vector of V slots a
// lane.  A group takes a token's heads one after another, q's and k's, so the
// token's cosines and sines are found once; sums over a head go across the
// group's lanes.  A lane writes the places of the values that it has read, and no
// others: outputs may be the inputs' own rows.
//
// Memory is the bound: 64 x 4,096 rows of 2 x 8 heads of 64, bfloat16, three
// quarters of them inside their sequences: norms 210 us (4.5 TB/s read and
// written), gradient 306 us (4.4 TB/s), one after the other 518.  One token of 512
// requests: 5.1 us, mostly the launch.
#include "nsfps_launch.h"
#include "nsfps_seq_device.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

struct NormDev {
  uint32_t length, q_heads, k_heads, head_dim, rotary_dim;
  uint32_t half;             // slots of rotated pairs, then of pairs behind them
  uint32_t rest;
  uint32_t lanes;            // of a group
  uint32_t per, chunks;      // heads of an item, items of a token
  uint32_t neighbours;
  float eps;
  uint64_t items;            // tokens * chunks
  nsfps_rows q, k, q_out, k_out;  // gradient: x and dx (q_out: dq)
  nsfps_rows dq_out, dk_out;      // gradient only
  const void *q_weight, *k_weight;
  const float *freq;
  const int32_t *lengths, *positions;
};

// The place of this lane's slots in a head, and which of them exist.
template <int V>
struct Slots {
  uint32_t first, second;  // elements of the first slot's two values
  uint32_t step;           // elements from slot to slot (2 where pairs are neighbours)
  bool one, two;           // whether the slots have a first and a second value
};
template <int V>
__device__ __forceinline__ Slots<V> slots_at(const NormDev &a, uint32_t s) {
  Slots<V> o;
  const bool turned = s < a.half;
  o.one = s < a.half + a.rest;
  o.step = 1;
  if (turned && a.neighbours) {
    o.first = 2 * s;
    o.second = V == 1 ? 2 * s + 1 : 2 * s + V;  // V slots are 2 V values in a row
  } else if (turned) {
    o.first = s;
    o.second = s + a.half;
  } else {
    o.first = a.rotary_dim + (s - a.half);
    o.second = o.first + a.rest;
  }
  o.two = o.one && o.second < a.head_dim;
  return o;
}

// Values of the slots: a (first of each pair) and b.
template <typename T, int V>
struct RawPair {
  Raw<T, V> a, b;
};
template <typename T, int V>
__device__ __forceinline__ RawPair<T, V> load_pair(const T *head, const Slots<V> &s) {
  RawPair<T, V> o{zero_raw<T, V>(), zero_raw<T, V>()};
  if (s.one) o.a = load_raw<T, V>(head + s.first);
  if (s.two) o.b = load_raw<T, V>(head + s.second);
  return o;
}
// neighbours: 2 V values in a row are V pairs
template <int V>
__device__ __forceinline__ void part(bool neighbours, float (&a)[V], float (&b)[V]) {
  if constexpr (V > 1) {
    if (!neighbours) return;
    float e[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = a[i], e[V + i] = b[i];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = e[2 * i], b[i] = e[2 * i + 1];
  }
}
template <int V>
__device__ __forceinline__ void unpart(bool neighbours, float (&a)[V], float (&b)[V]) {
  if constexpr (V > 1) {
    if (!neighbours) return;
    float e[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[2 * i] = a[i], e[2 * i + 1] = b[i];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = e[i], b[i] = e[V + i];
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_pair(T *head, const Slots<V> &s, const float (&a)[V],
                                           const float (&b)[V]) {
  if (s.one) store_f32<T, V>(head + s.first, a);
  if (s.two) store_f32<T, V>(head + s.second, b);
}

// Cosine and sine of position * freq.  Whole turns drop out, so what counts is the
// angle's error in radians: with products in float64 alone it was 2^-20 at the farthest
// position and freq 1, 2^-10 at freq 1,000.  Therefore angle and 1 / (2 pi) are two
// float64 each, and the turns the sum of their products' parts: off by 2^-32 radians at
// freq 2^40, less below, beside the 2^-23 that float32 leaves of half a turn.  (The
// norms of the case above take as long with either.)
__device__ __forceinline__ void turn(double position, float freq, float &c, float &s) {
#pragma clang fp contract(off)
  constexpr double kTurn = 0x1.45f306dc9c883p-3, kLow = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
  const double f = (double)freq, angle = position * f, rest = fma(position, f, -angle);
  const double turns = angle * kTurn;
  double t = (turns - rint(turns)) + (fma(angle, kTurn, -turns) + fma(angle, kLow, rest * kTurn));
  t -= rint(t);
  sincospif(2.f * (float)t, &s, &c);
}

__device__ __forceinline__ float group_sum(float v, uint32_t lanes) {
  for (uint32_t off = lanes / 2; off; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// A token's place, and its angles for this lane's slots (found while its first
// head's values are on their way).
template <int V, int S>
struct Token {
  uint32_t b, t;
  bool inside;
  float c[S][V], s[S][V];
};
template <int V, int S>
__device__ __forceinline__ void token_at(const NormDev &a, uint32_t token, Token<V, S> &o) {
  o.b = token / a.length;
  o.t = token % a.length;
  o.inside = true;
  if (a.lengths) {
    const int32_t n = a.lengths[o.b];
    o.inside = n > 0 && o.t < (uint32_t)n;
  }
}
// This lane's frequencies, 0 behind the rotation: cosine 1 and sine 0.
template <int V, int S>
__device__ __forceinline__ void load_freq(const NormDev &a, uint32_t lane, float (&f)[S][V]) {
  struct __attribute__((packed, aligned(4))) Some {
    float v[V];
  };
#pragma unroll
  for (int q = 0; q < S; ++q) {
    const uint32_t s0 = V * (lane + q * a.lanes);  // V slots are all turned or none
#pragma unroll
    for (int i = 0; i < V; ++i) f[q][i] = 0.f;
    if (s0 < a.half) {
      const Some o = *(const NSFPS_GLOBAL_SEQ Some *)(a.freq + s0);
#pragma unroll
      for (int i = 0; i < V; ++i) f[q][i] = o.v[i];
    }
  }
}
template <int V, int S>
__device__ __forceinline__ void find_angles(const NormDev &a, const float (&f)[S][V],
                                            Token<V, S> &o) {
  const int32_t from = a.positions ? max(a.positions[o.b], 0) : 0;
  const double position = (double)((int64_t)from + o.t);
#pragma unroll
  for (int q = 0; q < S; ++q)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o.c[q][i] = 1.f, o.s[q][i] = 0.f;
      if (a.half) turn(position, f[q][i], o.c[q][i], o.s[q][i]);
    }
}

template <typename T, int V, int S>
__device__ __forceinline__ void load_head_weights(const NormDev &a, const void *weight,
                                                  uint32_t lane, float (&wa)[S][V],
                                                  float (&wb)[S][V]) {
#pragma unroll
  for (int q = 0; q < S; ++q) {
    const Slots<V> s = slots_at<V>(a, V * (lane + q * a.lanes));
#pragma unroll
    for (int i = 0; i < V; ++i) wa[q][i] = wb[q][i] = 1.f;
    if (weight) {
      const RawPair<T, V> w = load_pair<T, V>((const T *)weight, s);
      numbers<T, V>(w.a, wa[q]);
      numbers<T, V>(w.b, wb[q]);
    }
    part<V>(a.neighbours && V * (lane + q * a.lanes) < a.half, wa[q], wb[q]);
  }
}

template <typename T>
__device__ __forceinline__ T *head_at(const NormDev &a, const nsfps_rows &q, const nsfps_rows &k,
                                      uint32_t b, uint32_t t, uint32_t h) {
  const bool is_k = h >= a.q_heads;
  const nsfps_rows &r = is_k ? k : q;
  return (T *)r.p + (uint64_t)b * r.batch_stride + (uint64_t)t * r.row_stride +
         (uint64_t)(is_k ? h - a.q_heads : h) * a.head_dim;
}

template <typename T, int V, int S>
__global__ __launch_bounds__(256) void k_norm(NormDev a) {
  const uint32_t lane = threadIdx.x % a.lanes, groups = 256 / a.lanes;
  Slots<V> at[S];
  bool mixed[S];  // slots that are pairs of neighbours
#pragma unroll
  for (int q = 0; q < S; ++q) {
    const uint32_t s0 = V * (lane + q * a.lanes);
    at[q] = slots_at<V>(a, s0);
    mixed[q] = a.neighbours && s0 < a.half;
  }
  float freq[S][V], wqa[S][V], wqb[S][V], wka[S][V], wkb[S][V];
  load_freq<V, S>(a, lane, freq);
  load_head_weights<T, V, S>(a, a.q_weight, lane, wqa, wqb);
  load_head_weights<T, V, S>(a, a.k_weight, lane, wka, wkb);
  const uint32_t heads = a.q_heads + a.k_heads;
  const float inv = 1.f / (float)a.head_dim;
  for (uint64_t item = (uint64_t)blockIdx.x * groups + threadIdx.x / a.lanes; item < a.items;
       item += (uint64_t)gridDim.x * groups) {
    const uint32_t h0 = (uint32_t)(item % a.chunks) * a.per, h1 = min(h0 + a.per, heads);
    Token<V, S> tok;
    token_at<V, S>(a, (uint32_t)(item / a.chunks), tok);
    RawPair<T, V> next[S];
    const auto fetch = [&](uint32_t h) {
      const T *x = head_at<const T>(a, a.q, a.k, tok.b, tok.t, h);
#pragma unroll
      for (int q = 0; q < S; ++q) next[q] = load_pair<T, V>(x, at[q]);
    };
    if (tok.inside) {
      fetch(h0);
      find_angles<V, S>(a, freq, tok);
    }
    for (uint32_t h = h0; h < h1; ++h) {
      T *const y = head_at<T>(a, a.q_out, a.k_out, tok.b, tok.t, h);
      float xa[S][V], xb[S][V];
      if (!tok.inside) {
#pragma unroll
        for (int q = 0; q < S; ++q) {
#pragma unroll
          for (int i = 0; i < V; ++i) xa[q][i] = xb[q][i] = 0.f;
          store_pair<T, V>(y, at[q], xa[q], xb[q]);
        }
        continue;
      }
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < S; ++q) {
        numbers<T, V>(next[q].a, xa[q]);
        numbers<T, V>(next[q].b, xb[q]);
        part<V>(mixed[q], xa[q], xb[q]);
      }
      if (h + 1 < h1) fetch(h + 1);
#pragma unroll
      for (int q = 0; q < S; ++q)
#pragma unroll
        for (int i = 0; i < V; ++i)
          sum = fmaf(xa[q][i], xa[q][i], fmaf(xb[q][i], xb[q][i], sum));
      const float r = rsqrtf(fmaf(group_sum(sum, a.lanes), inv, a.eps));
      const bool is_k = h >= a.q_heads;
#pragma unroll
      for (int q = 0; q < S; ++q) {
        float ya[V], yb[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = xa[q][i] * r * (is_k ? wka[q][i] : wqa[q][i]),
                      v = xb[q][i] * r * (is_k ? wkb[q][i] : wqb[q][i]);
          ya[i] = u * tok.c[q][i] - v * tok.s[q][i];
          yb[i] = u * tok.s[q][i] + v * tok.c[q][i];
        }
        unpart<V>(mixed[q], ya, yb);
        store_pair<T, V>(y, at[q], ya, yb);
      }
    }
  }
}

// The weights' sums stay in registers over a group's items, of kTerms heads at most
// (norm_blocks), so that a sum is off by kTerms 2^-24 of its terms' sizes whatever the
// tokens; they are added in a workgroup through LDS in the groups' order, and
// k_norm_join adds the workgroups' sums in theirs, both in float64.  parts:
// [workgroups][2][head_dim].
template <typename T, int V, int S>
__global__ __launch_bounds__(256) void k_norm_grad(NormDev a, float *__restrict__ parts) {
  __shared__ float s_sum[256 * 2 * S * V];
  const uint32_t lane = threadIdx.x % a.lanes, groups = 256 / a.lanes, d = a.head_dim;
  Slots<V> at[S];
  bool mixed[S];
#pragma unroll
  for (int q = 0; q < S; ++q) {
    const uint32_t s0 = V * (lane + q * a.lanes);
    at[q] = slots_at<V>(a, s0);
    mixed[q] = a.neighbours && s0 < a.half;
  }
  float freq[S][V], wqa[S][V], wqb[S][V], wka[S][V], wkb[S][V];
  load_freq<V, S>(a, lane, freq);
  load_head_weights<T, V, S>(a, a.q_weight, lane, wqa, wqb);
  load_head_weights<T, V, S>(a, a.k_weight, lane, wka, wkb);
  float qa[S][V] = {}, qb[S][V] = {}, ka[S][V] = {}, kb[S][V] = {};
  const uint32_t heads = a.q_heads + a.k_heads;
  const float inv = 1.f / (float)d;
  for (uint64_t item = (uint64_t)blockIdx.x * groups + threadIdx.x / a.lanes; item < a.items;
       item += (uint64_t)gridDim.x * groups) {
    const uint32_t h0 = (uint32_t)(item % a.chunks) * a.per, h1 = min(h0 + a.per, heads);
    Token<V, S> tok;
    token_at<V, S>(a, (uint32_t)(item / a.chunks), tok);
    RawPair<T, V> nx[S], ng[S];
    const auto fetch = [&](uint32_t h) {
      const T *x = head_at<const T>(a, a.q, a.k, tok.b, tok.t, h);
      const T *g = head_at<const T>(a, a.dq_out, a.dk_out, tok.b, tok.t, h);
#pragma unroll
      for (int q = 0; q < S; ++q) {
        nx[q] = load_pair<T, V>(x, at[q]);
        ng[q] = load_pair<T, V>(g, at[q]);
      }
    };
    if (tok.inside) {
      fetch(h0);
      find_angles<V, S>(a, freq, tok);
    }
    for (uint32_t h = h0; h < h1; ++h) {
      T *const dx = head_at<T>(a, a.q_out, a.k_out, tok.b, tok.t, h);
      float xa[S][V], xb[S][V], ga[S][V], gb[S][V];
      if (!tok.inside) {
#pragma unroll
        for (int q = 0; q < S; ++q) {
#pragma unroll
          for (int i = 0; i < V; ++i) xa[q][i] = xb[q][i] = 0.f;
          store_pair<T, V>(dx, at[q], xa[q], xb[q]);
        }
        continue;
      }
#pragma unroll
      for (int q = 0; q < S; ++q) {
        numbers<T, V>(nx[q].a, xa[q]);
        numbers<T, V>(nx[q].b, xb[q]);
        numbers<T, V>(ng[q].a, ga[q]);
        numbers<T, V>(ng[q].b, gb[q]);
        part<V>(mixed[q], xa[q], xb[q]);
        part<V>(mixed[q], ga[q], gb[q]);
      }
      if (h + 1 < h1) fetch(h + 1);
      const bool is_k = h >= a.q_heads;
      float squares = 0.f, along = 0.f;  // sums of x^2 and of g w x
#pragma unroll
      for (int q = 0; q < S; ++q)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = ga[q][i] * tok.c[q][i] + gb[q][i] * tok.s[q][i];
          const float v = gb[q][i] * tok.c[q][i] - ga[q][i] * tok.s[q][i];
          ga[q][i] = u, gb[q][i] = v;
          squares = fmaf(xa[q][i], xa[q][i], fmaf(xb[q][i], xb[q][i], squares));
          along = fmaf(u * (is_k ? wka[q][i] : wqa[q][i]), xa[q][i],
                       fmaf(v * (is_k ? wkb[q][i] : wqb[q][i]), xb[q][i], along));
        }
      const float r = rsqrtf(fmaf(group_sum(squares, a.lanes), inv, a.eps));
      // (a head whose squares pass float32 has a root of 0, and all of it is 0, though
      // the other sum may have passed float32 too)
      const float dot = group_sum(along, a.lanes), back = r > 0.f ? dot * inv * r * r : 0.f;
#pragma unroll
      for (int q = 0; q < S; ++q) {
        float da[V], db[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float sa = ga[q][i] * (xa[q][i] * r), sb = gb[q][i] * (xb[q][i] * r);
          qa[q][i] += is_k ? 0.f : sa, qb[q][i] += is_k ? 0.f : sb;
          ka[q][i] += is_k ? sa : 0.f, kb[q][i] += is_k ? sb : 0.f;
          da[i] = r * (ga[q][i] * (is_k ? wka[q][i] : wqa[q][i]) - xa[q][i] * back);
          db[i] = r * (gb[q][i] * (is_k ? wkb[q][i] : wqb[q][i]) - xb[q][i] * back);
        }
        unpart<V>(mixed[q], da, db);
        store_pair<T, V>(dx, at[q], da, db);
      }
    }
  }
  for (int side = 0; side < 2; ++side) {
    __syncthreads();
    float *const mine = s_sum + threadIdx.x / a.lanes * d;
#pragma unroll
    for (int q = 0; q < S; ++q) {
      float va[V], vb[V];
#pragma unroll
      for (int i = 0; i < V; ++i)
        va[i] = side ? ka[q][i] : qa[q][i], vb[i] = side ? kb[q][i] : qb[q][i];
      unpart<V>(mixed[q], va, vb);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (at[q].one) mine[at[q].first + i] = va[i];
        if (at[q].two) mine[at[q].second + i] = vb[i];
      }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < d; e += 256) {
      double sum = 0.;
      for (uint32_t g = 0; g < groups; ++g) sum += s_sum[g * d + e];
      parts[((uint64_t)blockIdx.x * 2 + side) * d + e] = (float)sum;
    }
  }
}

// 8 values and 32 runs of workgroups a workgroup, eight loads of a run together:
// 5.4 us for 1,024 workgroups' sums of 64 values.
__global__ __launch_bounds__(256) void k_norm_join(const float *__restrict__ parts, uint32_t blocks,
                                                   uint32_t d, float *dq_weight, float *dk_weight) {
  constexpr uint32_t kRuns = 32, kAhead = 8;
  __shared__ double s_sum[kRuns][8];
  const uint32_t side = blockIdx.y, e = blockIdx.x * 8 + threadIdx.x % 8, run = threadIdx.x / 8;
  float *const out = side ? dk_weight : dq_weight;
  double sum = 0.;
  if (e < d)
    for (uint32_t b = run; b < blocks; b += kRuns * kAhead) {
      float v[kAhead];
#pragma unroll
      for (uint32_t k = 0; k < kAhead; ++k)
        v[k] = parts[((uint64_t)min(b + kRuns * k, blocks - 1) * 2 + side) * d + e];
#pragma unroll
      for (uint32_t k = 0; k < kAhead; ++k) sum += b + kRuns * k < blocks ? v[k] : 0.f;
    }
  s_sum[run][threadIdx.x % 8] = sum;
  __syncthreads();
  if (threadIdx.x < 8 && e < d && out) {
    double all = 0.;
    for (uint32_t k = 0; k < kRuns; ++k) all += s_sum[k][threadIdx.x];
    out[e] = (float)all;
  }
}

constexpr uint32_t kGradBlocks = 1024;
constexpr uint32_t kTerms = 256;  // heads that a lane adds one after another

NormDev norm_dev(const nsfps_norm_args &a) {
  NormDev d = {};
  d.length = (uint32_t)a.length;
  d.q_heads = a.q_heads;
  d.k_heads = a.k_heads;
  d.head_dim = a.head_dim;
  d.rotary_dim = a.rotary_dim;
  d.half = a.rotary_dim / 2;
  d.rest = (a.head_dim - a.rotary_dim + 1) / 2;
  d.neighbours = a.neighbours != 0;
  d.eps = a.eps;
  d.q = a.q;
  d.k = a.k;
  d.q_out = a.q_out;
  d.k_out = a.k_out;
  d.q_weight = a.d_q_weight;
  d.k_weight = a.d_k_weight;
  d.freq = a.d_freq;
  d.lengths = a.d_lengths;
  d.positions = a.d_positions;
  return d;
}

// Slots of a vector: as many as the rotation, the head and every address keep
// aligned, at most 16 bytes (us of norms and gradient of the case above: 518 with 8
// bfloat16 values, 1,366 with single ones).
uint32_t norm_vector(const nsfps_norm_args &a, std::initializer_list<const nsfps_rows *> rows) {
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2;
  const uint32_t half = a.rotary_dim / 2, behind = a.head_dim - a.rotary_dim;
  uint32_t v = 16 / size;
  const auto fits = [&](uint32_t n) {
    if (half % n || behind % (2 * n) || a.head_dim % n) return false;
    if (((uintptr_t)a.d_q_weight | (uintptr_t)a.d_k_weight) % (n * size)) return false;
    for (const nsfps_rows *r : rows)
      if ((uintptr_t)r->p % (n * size) || (a.batch > 1 && r->batch_stride % n) ||
          (a.length > 1 && r->row_stride % n))
        return false;
    return true;
  };
  while (v > 1 && !fits(v)) v /= 2;
  return v;
}

void norm_split(NormDev &d, uint64_t tokens, uint32_t v, uint32_t most = ~0u) {
  const uint32_t slots = d.half + d.rest;
  uint32_t lanes = 1;
  while (lanes < 64 && lanes * v < slots) lanes *= 2;
  d.lanes = lanes;
  // heads of an item: all, so that a token's angles, in float64, are found once (us of
  // norms and gradient of the case above 518, 831 with a head an item), unless tokens
  // are too few to fill the chip (a call of one token of 64 + 64 heads of 128: 9.7,
  // 125 with all heads an item)
  constexpr uint64_t kFill = 256 * 1024;  // threads
  const uint32_t heads = d.q_heads + d.k_heads;
  const uint64_t want = std::max<uint64_t>(host_ceil_div(heads, most),
                                           kFill / std::max<uint64_t>(1, tokens * lanes));
  d.chunks = (uint32_t)std::min<uint64_t>(heads, want);
  d.per = (heads + d.chunks - 1) / d.chunks;
  d.chunks = (heads + d.per - 1) / d.per;
  d.items = tokens * d.chunks;
}

template <typename F>
hipError_t norm_by(uint32_t dtype, uint32_t v, uint32_t slots, F f) {
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, 4> four;
  constexpr std::integral_constant<int, 8> eight;
  const auto by_vector = [&](auto t) {
    if constexpr (sizeof(t) == 2)
      if (v == 8) return f(t, eight, one);
    if (v == 4) return f(t, four, one);
    if (v == 2) return f(t, two, one);
    return slots <= 64 ? f(t, one, one) : f(t, one, two);
  };
  return dtype == NSFPS_F32 ? by_vector(float()) : by_vector(bf16());
}

uint32_t norm_grid(const NormDev &d, uint64_t most) {
  return (uint32_t)std::min<uint64_t>(most, host_ceil_div(d.items, 256 / d.lanes));
}

// Workgroups of the gradient: kGradBlocks at most, or as many as leave a group kTerms
// heads (an item has no more of them, by norm_split).  us of norms and gradient of
// 16 x 65,536 rows of 8 + 8 heads of 64 bfloat16, single values: 4,739 so, 5,623 with
// kGradBlocks alone; of 64 x 16,384 in vectors, where kGradBlocks are enough, 2,092.
uint64_t norm_blocks(const NormDev &d) {
  const uint64_t groups = 256 / d.lanes, items = std::max<uint64_t>(1, kTerms / d.per);
  return std::max(std::min<uint64_t>(kGradBlocks, host_ceil_div(d.items, groups)),
                  host_ceil_div(d.items, groups * items));
}

}  // namespace

hipError_t launch_norm(const nsfps_norm_args &a, hipStream_t st) {
  NormDev d = norm_dev(a);
  nsfps_rows none = {};
  const nsfps_rows *q = a.q_heads ? &a.q : &none, *qo = a.q_heads ? &a.q_out : &none,
                   *k = a.k_heads ? &a.k : &none, *ko = a.k_heads ? &a.k_out : &none;
  const uint32_t v = norm_vector(a, {q, qo, k, ko});
  norm_split(d, a.batch * a.length, v);
  return norm_by(a.dtype, v, d.half + d.rest, [&](auto t, auto vec, auto sets) {
    k_norm<decltype(t), decltype(vec)::value, decltype(sets)::value>
        <<<norm_grid(d, 1u << 20), 256, 0, st>>>(d);
    return hipGetLastError();
  });
}

// Of whichever vector the rows' addresses allow.
uint64_t norm_grad_bytes(const nsfps_norm_args &a) {
  uint64_t blocks = kGradBlocks;
  for (uint32_t v = 1; v <= 8; v *= 2) {
    NormDev d = norm_dev(a);
    norm_split(d, a.batch * a.length, v, kTerms);
    blocks = std::max(blocks, norm_blocks(d));
  }
  return 4 * blocks * 2 * a.head_dim;
}

hipError_t launch_norm_grad(const nsfps_norm_args &a, const nsfps_norm_grads &g, hipStream_t st) {
  NormDev d = norm_dev(a);
  d.q_out = g.dq;
  d.k_out = g.dk;
  d.dq_out = g.dq_out;
  d.dk_out = g.dk_out;
  nsfps_rows none = {};
  const bool q = a.q_heads != 0, k = a.k_heads != 0;
  const uint32_t v = norm_vector(a, {q ? &a.q : &none, q ? &g.dq : &none, q ? &g.dq_out : &none,
                                     k ? &a.k : &none, k ? &g.dk : &none, k ? &g.dk_out : &none});
  norm_split(d, a.batch * a.length, v, kTerms);
  const uint32_t blocks = (uint32_t)norm_blocks(d);
  float *const parts = (float *)a.workspace;
  hipError_t e = hipSuccess;
  if (blocks)
    e = norm_by(a.dtype, v, d.half + d.rest, [&](auto t, auto vec, auto sets) {
      k_norm_grad<decltype(t), decltype(vec)::value, decltype(sets)::value>
          <<<blocks, 256, 0, st>>>(d, parts);
      return hipGetLastError();
    });
  if (e != hipSuccess || (!g.d_dq_weight && !g.d_dk_weight)) return e;
  k_norm_join<<<dim3((a.head_dim + 7) / 8, 2), 256, 0, st>>>(parts, blocks, a.head_dim,
                                                              g.d_dq_weight, g.d_dk_weight);
  return hipGetLastError();
}

hipError_t preload_norm_kernels() {
  return func_attributes(k_norm<bf16, 8, 1>, k_norm_grad<bf16, 8, 1>, k_norm_join);
}

}  // namespace nsfps
