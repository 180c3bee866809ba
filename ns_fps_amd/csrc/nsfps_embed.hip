// Embedding lookup with scaling, and its gradient by sorted tokens.
//
// Lookup: out[i] = scale * table[tok[i]].  Each row is read and written once,
// in 16-byte pieces where the rows are aligned; memory is the bound.
//
// Gradient: dtable[v] = scale * sum of dout[i] over tok[i] = v.  The tokens
// are sorted with their positions (stable, so a row's positions are in
// order), start[v] is found at the sorted tokens' boundaries, and one wave
// per table row adds that row's terms in float32, in that order, and writes
// the row once: no atomics on values, the same bits every time, and rows
// without a token cost their zeros.  A crowded row (more than kLong terms:
// grid cells near an object) is cut into pieces of kPiece terms, a wave each,
// whose sums (in float64: the
// terms may be many) are added in order by a last pass.  Where pieces lie in the
// workspace is decided by an atomic counter; no sum depends on it.
#include "nsfps_launch.h"
#include "nsfps_seq_device.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

constexpr uint32_t kLong = 64;    // terms of one wave's row
constexpr uint32_t kPiece = 256;  // terms of a piece of a longer one

// Workgroups of a grid-stride kernel: a launch holds fewer than 2^32 threads.
uint32_t grid_of(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, 1u << 20); }

// ---- lookup

// tpr threads (a power of two, at most 256) per row, V elements each
template <typename T, int V>
__global__ __launch_bounds__(256) void k_embed(const T *__restrict__ table,
                                               const int32_t *__restrict__ tokens,
                                               T *__restrict__ out, uint32_t count, uint32_t rows,
                                               uint32_t vecs, uint64_t table_stride,
                                               uint64_t out_stride, float scale, uint32_t tpr) {
  const uint32_t per = 256 / tpr;
  for (uint64_t i = (uint64_t)blockIdx.x * per + threadIdx.x / tpr; i < count;
       i += (uint64_t)gridDim.x * per) {
    const int32_t tok = tokens[i];
    const bool hit = tok >= 0 && (uint32_t)tok < rows;
    const T *src = table + (hit ? (uint64_t)tok * table_stride : 0);
    T *dst = out + i * out_stride;
    for (uint32_t c = threadIdx.x % tpr; c < vecs; c += tpr) {
      float v[V];
      if (hit) {
        load_f32<T, V>(src + (uint64_t)c * V, v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] *= scale;
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = 0.f;
      }
      store_f32<T, V>(dst + (uint64_t)c * V, v);
    }
  }
}

// ---- gradient

// keys: the tokens, rows for those outside
__global__ __launch_bounds__(256) void k_embed_keys(const int32_t *__restrict__ tokens,
                                                    uint32_t count, uint32_t rows,
                                                    uint32_t *__restrict__ keys,
                                                    uint32_t *__restrict__ counters) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i < 2) counters[i] = 0;
  if (i >= count) return;
  const int32_t t = tokens[i];
  keys[i] = t >= 0 && (uint32_t)t < rows ? (uint32_t)t : rows;
}

// start[v] (v <= rows): sorted positions below it hold tokens below v.
// Position p = 0 .. count fills start over (key[p - 1], key[p]], key[-1] = -1
// and key[count] = rows; long gaps are filled by the whole workgroup.
__global__ __launch_bounds__(256) void k_embed_starts(const uint32_t *__restrict__ keys,
                                                      uint32_t count, uint32_t rows,
                                                      uint32_t *__restrict__ start) {
  __shared__ uint32_t s_n, s_lo[256], s_hi[256], s_p[256];
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  const uint64_t p = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (p <= count) {
    const uint32_t lo = p == 0 ? 0u : keys[p - 1] + 1, hi = p == count ? rows : keys[p];
    // entries lo .. hi (none where the token is the one before it, or both are outside)
    if (lo <= hi) {
      if (hi - lo < 16) {
        for (uint32_t v = lo; v <= hi; ++v) start[v] = (uint32_t)p;
      } else {
        const uint32_t k = atomicAdd(&s_n, 1u);
        s_lo[k] = lo;
        s_hi[k] = hi;
        s_p[k] = (uint32_t)p;
      }
    }
  }
  __syncthreads();
  const uint32_t n = s_n;
  for (uint32_t k = 0; k < n; ++k)
    for (uint64_t v = (uint64_t)s_lo[k] + threadIdx.x; v <= s_hi[k]; v += 256) start[v] = s_p[k];
}

// acc += the terms pos[from .. to) of one column vector, in order
template <typename T, int V, typename A>
__device__ __forceinline__ void add_terms(const T *__restrict__ dout, uint64_t stride,
                                          const uint32_t *__restrict__ pos, uint32_t from,
                                          uint32_t to, A (&acc)[V]) {
  constexpr uint32_t kAhead = 4;  // loads in flight
  uint32_t p = from;
  for (; p + kAhead <= to; p += kAhead) {
    float v[kAhead][V];
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j)
      load_f32<T, V>(dout + (uint64_t)pos[p + j] * stride, v[j]);
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += v[j][k];
  }
  for (; p < to; ++p) {
    float v[V];
    load_f32<T, V>(dout + (uint64_t)pos[p] * stride, v);
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += v[k];
  }
}

struct LongRow {
  uint32_t row, piece;  // the row, and its first piece in the workspace
};

// One wave per table row.  Crowded rows are listed: counters[0] counts them,
// counters[1] their pieces; piece_at[k] = the sorted position piece k starts at.
template <typename T, typename G, int V>
__global__ __launch_bounds__(256) void k_embed_rows(
    const T *__restrict__ dout, uint64_t dout_stride, const uint32_t *__restrict__ pos,
    const uint32_t *__restrict__ start, G *__restrict__ dtable, uint64_t table_stride,
    uint32_t rows, uint32_t vecs, float scale, uint32_t *__restrict__ counters,
    LongRow *__restrict__ longs, uint2 *__restrict__ piece_at) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows;
       row += (uint64_t)gridDim.x * 4) {
    const uint32_t from = start[row], to = start[row + 1];
    if (to - from > kLong) {
      const uint32_t pieces = ceil_div(to - from, kPiece);
      uint32_t first = 0;
      if (lane == 0) {
        first = atomicAdd(&counters[1], pieces);
        longs[atomicAdd(&counters[0], 1u)] = LongRow{(uint32_t)row, first};
      }
      first = __shfl(first, 0, 64);
      for (uint32_t k = lane; k < pieces; k += 64) {
        const uint32_t f = from + k * kPiece;
        piece_at[first + k] = make_uint2(f, f + min(kPiece, to - f));
      }
      continue;
    }
    G *dst = dtable + row * table_stride;
    for (uint32_t c = lane; c < vecs; c += 64) {
      float acc[V] = {};
      add_terms<T, V>(dout + (uint64_t)c * V, dout_stride, pos, from, to, acc);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] *= scale;
      store_f32<G, V>(dst + (uint64_t)c * V, acc);
    }
  }
}

// One wave per piece and 64 column vectors; part: pieces x width, in float64:
// a crowded row may have tens of thousands of terms
template <typename T, int V>
__global__ __launch_bounds__(64) void k_embed_pieces(const T *__restrict__ dout,
                                                     uint64_t dout_stride,
                                                     const uint32_t *__restrict__ pos,
                                                     const uint32_t *__restrict__ counters,
                                                     const uint2 *__restrict__ piece_at,
                                                     double *__restrict__ part, uint32_t vecs,
                                                     uint32_t width) {
  const uint32_t n = counters[1];
  const uint32_t c = blockIdx.y * 64 + threadIdx.x;
  if (c >= vecs) return;
  for (uint32_t k = blockIdx.x; k < n; k += gridDim.x) {
    const uint2 at = piece_at[k];
    double acc[V] = {};
    add_terms<T, V>(dout + (uint64_t)c * V, dout_stride, pos, at.x, at.y, acc);
#pragma unroll
    for (int j = 0; j < V; ++j) part[(uint64_t)k * width + c * V + j] = acc[j];
  }
}

// The crowded rows: 16 waves each add a run of a row's pieces, then the
// runs' sums are added in order.
template <typename G>
__global__ __launch_bounds__(1024) void k_embed_join(const uint32_t *__restrict__ counters,
                                                     const LongRow *__restrict__ longs,
                                                     const uint32_t *__restrict__ start,
                                                     const double *__restrict__ part,
                                                     G *__restrict__ dtable, uint64_t table_stride,
                                                     uint32_t width, float scale) {
  __shared__ double s_sum[16][64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t n = counters[0];
  const uint32_t c = blockIdx.y * 64 + lane;
  for (uint32_t k = blockIdx.x; k < n; k += gridDim.x) {
    const LongRow lr = longs[k];
    const uint32_t pieces = ceil_div(start[lr.row + 1] - start[lr.row], kPiece);
    const uint32_t run = ceil_div(pieces, 16);
    const uint32_t a = min(wave * run, pieces), b = min(a + run, pieces);
    double acc = 0.0;
    if (c < width)
      for (uint32_t p = a; p < b; ++p) acc += part[(uint64_t)(lr.piece + p) * width + c];
    s_sum[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < width) {
      double t = 0.0;
#pragma unroll
      for (int w = 0; w < 16; ++w) t += s_sum[w][lane];
      const float o[1] = {(float)(t * scale)};
      store_f32<G, 1>(dtable + (uint64_t)lr.row * table_stride + c, o);
    }
    __syncthreads();
  }
}

// ---- workspace of the gradient

struct GradPlan {
  uint64_t keys, vals, keys2, vals2, hist, scan, start, counters, longs, pieces, part, total;
  uint32_t long_max, piece_max;
  int bits;
};

GradPlan grad_plan(const nsfps_embed_args &a) {
  GradPlan p;
  uint64_t off = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t at = off;
    off = (off + bytes + 255) & ~255ull;
    return at;
  };
  p.bits = 1;
  while (p.bits < 32 && (a.rows >> p.bits)) ++p.bits;  // keys 0 .. rows
  p.long_max = (uint32_t)(a.tokens / (kLong + 1));
  p.piece_max = (uint32_t)(a.tokens / kPiece) + p.long_max;
  const uint64_t hist = radix_hist_len((uint32_t)a.tokens);
  p.keys = take(4 * a.tokens);
  p.vals = take(4 * a.tokens);
  p.keys2 = take(4 * a.tokens);
  p.vals2 = take(4 * a.tokens);
  p.hist = take(4 * hist);
  p.scan = take(4 * (uint64_t)scan_tmp_len((uint32_t)hist));
  p.start = take(4 * (a.rows + 1));
  p.counters = take(8);
  p.longs = take(sizeof(LongRow) * (uint64_t)p.long_max);
  p.pieces = take(8 * (uint64_t)p.piece_max);
  p.part = take(8ull * p.piece_max * a.width);
  p.total = off;
  return p;
}

template <typename T, typename G, int V>
hipError_t run_grad(const nsfps_embed_args &a, hipStream_t st) {
  const GradPlan p = grad_plan(a);
  char *const w = (char *)a.workspace;
  uint32_t *const counters = (uint32_t *)(w + p.counters), *const start = (uint32_t *)(w + p.start);
  const uint32_t count = (uint32_t)a.tokens, rows = (uint32_t)a.rows;
  uint32_t *keys = (uint32_t *)(w + p.keys), *pos = (uint32_t *)(w + p.vals);
  k_embed_keys<<<(uint32_t)host_ceil_div(std::max(count, 2u), 256), 256, 0, st>>>(
      a.d_tokens, count, rows, keys, counters);
  if (count) {
    const hipError_t e = launch_radix_sort(keys, pos, (uint32_t *)(w + p.keys2),
                                           (uint32_t *)(w + p.vals2), count, p.bits,
                                           (uint32_t *)(w + p.hist), (uint32_t *)(w + p.scan), true,
                                           &keys, &pos, st);
    if (e != hipSuccess) return e;
  }
  k_embed_starts<<<(uint32_t)host_ceil_div((uint64_t)count + 1, 256), 256, 0, st>>>(keys, count,
                                                                                   rows, start);
  const uint32_t vecs = a.width / V;
  const T *dout = (const T *)a.d_out;
  G *dtable = (G *)a.d_table;
  LongRow *const longs = (LongRow *)(w + p.longs);
  uint2 *const pieces = (uint2 *)(w + p.pieces);
  double *const part = (double *)(w + p.part);
  k_embed_rows<T, G, V><<<grid_of(host_ceil_div(rows, 4)), 256, 0, st>>>(
      dout, a.out_stride, pos, start, dtable, a.table_stride, rows, vecs, a.scale, counters, longs,
      pieces);
  if (p.long_max) {
    const dim3 gp(std::min(p.piece_max, 4096u), (uint32_t)host_ceil_div(vecs, 64));
    k_embed_pieces<T, V><<<gp, 64, 0, st>>>(dout, a.out_stride, pos, counters, pieces, part, vecs,
                                            a.width);
    const dim3 gj(std::min(p.long_max, 512u), (uint32_t)host_ceil_div(a.width, 64));
    k_embed_join<G><<<gj, 1024, 0, st>>>(counters, longs, start, part, dtable, a.table_stride,
                                         a.width, a.scale);
  }
  return hipGetLastError();
}

bool wide_table(const void *p, uint64_t stride, uint32_t width, uint32_t v, uint32_t size) {
  return (uintptr_t)p % (v * size) == 0 && stride % v == 0 && width % v == 0;
}

}  // namespace

hipError_t launch_embed(const nsfps_embed_args &a, hipStream_t st) {
  const auto go = [&](auto *t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int V = decltype(v)::value;
    const uint32_t vecs = a.width / V;
    uint32_t tpr = 1;
    while (tpr < 256 && tpr < vecs) tpr *= 2;
    k_embed<T, V><<<grid_of(host_ceil_div(a.tokens, 256 / tpr)), 256, 0, st>>>(
        (const T *)a.d_table, a.d_tokens, (T *)a.d_out, (uint32_t)a.tokens, (uint32_t)a.rows, vecs,
        a.table_stride, a.out_stride, a.scale, tpr);
    return hipGetLastError();
  };
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2, v = 16 / size;
  const bool wide = wide_table(a.d_table, a.table_stride, a.width, v, size) &&
                    wide_table(a.d_out, a.out_stride, a.width, v, size);
  if (a.dtype == NSFPS_F32)
    return wide ? go((float *)nullptr, std::integral_constant<int, 4>())
                : go((float *)nullptr, std::integral_constant<int, 1>());
  return wide ? go((bf16 *)nullptr, std::integral_constant<int, 8>())
              : go((bf16 *)nullptr, std::integral_constant<int, 1>());
}

uint64_t embed_grad_bytes(const nsfps_embed_args &a) { return grad_plan(a).total; }

hipError_t launch_embed_grad(const nsfps_embed_args &a, hipStream_t st) {
  const bool tf = a.dtype == NSFPS_F32, gf = a.grad_dtype == NSFPS_F32;
  const uint32_t ts = tf ? 4 : 2, gs = gf ? 4 : 2;
  // 4 elements a lane where both sides' rows allow it (8 to 16 bytes a load)
  const bool wide = wide_table(a.d_out, a.out_stride, a.width, 4, ts) &&
                    wide_table(a.d_table, a.table_stride, a.width, 4, gs);
  if (tf)
    return gf ? (wide ? run_grad<float, float, 4>(a, st) : run_grad<float, float, 1>(a, st))
              : (wide ? run_grad<float, bf16, 4>(a, st) : run_grad<float, bf16, 1>(a, st));
  return gf ? (wide ? run_grad<bf16, float, 4>(a, st) : run_grad<bf16, float, 1>(a, st))
            : (wide ? run_grad<bf16, bf16, 4>(a, st) : run_grad<bf16, bf16, 1>(a, st));
}

hipError_t preload_embed_kernels() {
  return func_attributes(k_embed<bf16, 8>, k_embed<bf16, 1>, k_embed<float, 4>, k_embed<float, 1>,
                         k_embed_keys, k_embed_starts, k_embed_rows<bf16, bf16, 4>,
                         k_embed_rows<float, float, 4>);
}

}  // namespace nsfps
