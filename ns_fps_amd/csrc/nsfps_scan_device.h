// Pieces shared by the selective scan and its gradient: the chunk's steps and
// decays, the chunks' states, and the launch parameters.
#pragma once

#include "nsfps_mfma.h"

#pragma clang fp contract(fast)

namespace nsfps {
namespace seq {

constexpr uint32_t kChunk = 64;  // tokens of a chunk: four 16-row tiles, one per wave
constexpr uint32_t kPTile = 64;  // head_dim columns of a workgroup

// A call's sizes and inputs, as the kernels see them.
struct ScanDev {
  uint32_t batch, length, heads, groups, head_dim, state_dim;
  uint32_t chunks, ptiles;  // of the longest sequence; of head_dim
  nsfps_rows x, b, c, dt, y;
  const float *a, *d, *dt_bias;
  const int32_t *lengths, *positions, *slots;
  float *state;       // the cache, or null
  float *states;      // [batch][heads][chunks][head_dim][state_dim]
  float *totals;      // [batch][heads][chunks]: log2 of a whole chunk's decay
  uint32_t wide_x, wide_bc, wide_y;  // 16-byte accesses fit
};

__device__ __forceinline__ uint32_t scan_length(const ScanDev &s, uint32_t b) {
  if (!s.lengths) return s.length;
  const int32_t n = s.lengths[b];
  return n < 0 ? 0u : min((uint32_t)n, s.length);
}

// Steps of a chunk: delta, and s = the inclusive sum of delta * a in log2
// units as hi + lo, so that the difference of two sums keeps its own relative
// precision however far the chunk has decayed (a single float32 sum of -500
// would leave 3e-5 in the exponent of a decay near 1).
struct Steps {
  float delta[kChunk], hi[kChunk], lo[kChunk];
};

__device__ __forceinline__ float decay_between(const Steps &s, int i, int j) {  // j <= i
  return exp2_fast((s.hi[i] - s.hi[j]) + (s.lo[i] - s.lo[j]));
}

// The raw step of a token (before softplus), 0 steps past the sequence's end.
template <typename T>
__device__ __forceinline__ float raw_step(const ScanDev &s, uint32_t b, uint32_t h, uint32_t t) {
  float v[1];
  load_f32<T, 1>((const T *)s.dt.p + (uint64_t)b * s.dt.batch_stride +
                     (uint64_t)t * s.dt.row_stride + h, v);
  return v[0] + (s.dt_bias ? s.dt_bias[h] : 0.f);
}

// One wave fills the steps of chunk tokens t0 .. t0+63.
template <typename T>
__device__ __forceinline__ void chunk_steps(const ScanDev &s, Steps &o, uint32_t b, uint32_t h,
                                            uint32_t t0, uint32_t len) {
  const uint32_t lane = threadIdx.x & 63u;
  float delta = 0.f;
  if (t0 + lane < len) delta = softplus(raw_step<T>(s, b, h, t0 + lane));
  double sum = (double)delta * (double)s.a[h] * 1.4426950408889634074;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double o2 = __shfl_up(sum, off, 64);
    if (lane >= (uint32_t)off) sum += o2;
  }
  // below 2^-4096 every decay is 0 already; the bound keeps infinities out
  sum = fmax(sum, -1e30);
  o.delta[lane] = delta;
  o.hi[lane] = (float)sum;
  o.lo[lane] = (float)(sum - (double)(float)sum);
}

// Chunk sums: out[p][n] = sum over the chunk's tokens of weight * u[p] * v[n].
// Forward: u = x, v = b, weight = delta_j * decay from j to the chunk's end;
// reversed: u = dy, v = c, weight = decay from the chunk's start through i.
// The weighted u is split into three bfloat16 terms: the states are float32
// and keep float32 accuracy.
template <typename T, int NT, bool REV>
__global__ __launch_bounds__(256) void k_scan_sums(ScanDev s, nsfps_rows u, nsfps_rows v,
                                                   uint32_t wide_u, uint32_t wide_v,
                                                   float *__restrict__ states, uint64_t work) {
  constexpr int ldu = kLd<T, (int)kPTile>, ldv = kLd<T, NT>;
  __shared__ __attribute__((aligned(16))) T s_u[kChunk * ldu];
  __shared__ __attribute__((aligned(16))) T s_v[kChunk * ldv];
  __shared__ Steps s_st;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, l = lane & 15u;
  for (uint64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const uint32_t hp = (uint32_t)(w % (s.heads * s.ptiles));
    const uint64_t bc = w / (s.heads * s.ptiles);
    const uint32_t h = hp / s.ptiles, p0 = (hp % s.ptiles) * kPTile;
    const uint32_t c = (uint32_t)(bc % s.chunks), b = (uint32_t)(bc / s.chunks);
    const uint32_t len = scan_length(s, b), t0 = c * kChunk;
    if (t0 >= len) continue;
    const uint32_t rows = min(kChunk, len - t0), grp = h / (s.heads / s.groups);
    load_tile<T, (int)kPTile>(s_u, (const T *)u.p + (uint64_t)b * u.batch_stride +
                                       (uint64_t)t0 * u.row_stride + h * s.head_dim + p0,
                              u.row_stride, rows, s.head_dim - p0, wide_u);
    load_tile<T, NT>(s_v, (const T *)v.p + (uint64_t)b * v.batch_stride +
                              (uint64_t)t0 * v.row_stride + grp * s.state_dim,
                     v.row_stride, rows, s.state_dim, wide_v);
    if (wave == 0) chunk_steps<T>(s, s_st, b, h, t0, len);
    __syncthreads();
    f32x4 sum[NT / 16] = {}, low[NT / 16] = {};  // of the first terms; of the others
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      Terms<T, 3> ut[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int j = 32 * kk + 16 * half + 4 * g;
        f32x4 q = quad_f32(quad_col<T>(s_u, ldu, j, 16 * wave + l));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q[i] *= REV ? exp2_fast(s_st.hi[j + i] + s_st.lo[j + i])
                      : s_st.delta[j + i] * decay_between(s_st, kChunk - 1, j + i);
        ut[half] = split<T, 3>(q);
      }
#pragma unroll
      for (int nt = 0; nt < NT / 16; ++nt) {
        const Quad<T> a0 = quad_col<T>(s_v, ldv, 32 * kk + 4 * g, 16 * nt + l);
        const Quad<T> a1 = quad_col<T>(s_v, ldv, 32 * kk + 16 + 4 * g, 16 * nt + l);
#pragma unroll
        for (int i = Terms<T, 3>::kN - 1; i > 0; --i) mma(low[nt], a0, a1, ut[0].q[i], ut[1].q[i]);
        mma_apart(sum[nt], a0, a1, ut[0].q[0], ut[1].q[0]);
      }
    }
    const uint32_t p = p0 + 16 * wave + l;
    const uint64_t at = (uint64_t)b * s.heads * s.chunks + (uint64_t)h * s.chunks + c;
    float *out = states + (at * s.head_dim + p) * s.state_dim;
    if (p < s.head_dim) {
#pragma unroll
      for (int nt = 0; nt < NT / 16; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * nt + 4 * g + i < s.state_dim) out[16 * nt + 4 * g + i] = sum[nt][i] + low[nt][i];
    }
    if (!REV && p0 == 0 && threadIdx.x == 0) s.totals[at] = s_st.hi[kChunk - 1] + s_st.lo[kChunk - 1];
    __syncthreads();
  }
}

// The chunks' sums become the states at the chunks' starts (forward) or the
// states' gradients at the chunks' ends (reversed), in place; one thread per
// state value walks the sequence's chunks, kRun of them loaded ahead.
template <bool REV>
__global__ __launch_bounds__(256) void k_scan_pass(ScanDev s, float *__restrict__ states,
                                                   uint64_t values) {
  constexpr uint32_t kRun = 8;
  const uint32_t pn = s.head_dim * s.state_dim;
  for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < values;
       e += (uint64_t)gridDim.x * 256) {
    const uint64_t bh = e / pn;
    const uint32_t b = (uint32_t)(bh / s.heads), at = (uint32_t)(e % pn);
    const uint32_t n = (scan_length(s, b) + kChunk - 1) / kChunk;
    float run = 0.f;
    float *cache = nullptr;
    if (!REV && s.state) {
      const int32_t slot = s.slots ? s.slots[b] : (int32_t)b;
      if (slot >= 0) {
        cache = s.state + ((uint64_t)slot * s.heads + bh % s.heads) * pn + at;
        if (s.positions && s.positions[b] > 0) run = *cache;
      }
    }
    float *st = states + bh * s.chunks * pn + at;
    const float *tot = s.totals + bh * s.chunks;
    for (uint32_t c0 = 0; c0 < n; c0 += kRun) {
      float v[kRun], t[kRun];
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) {
        const uint32_t i = min(c0 + k, n - 1), c = REV ? n - 1 - i : i;
        v[k] = st[(uint64_t)c * pn];
        t[k] = tot[c];
      }
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) {
        if (c0 + k >= n) break;
        const uint32_t c = REV ? n - 1 - (c0 + k) : c0 + k;
        st[(uint64_t)c * pn] = run;
        run = fmaf(exp2_fast(t[k]), run, v[k]);
      }
    }
    if (cache && n) *cache = run;
  }
}

inline uint32_t scan_grid(uint64_t work, uint64_t most = 1u << 20) {
  return (uint32_t)(work < most ? work : most);
}

// Bytes of one launch's chunk states and totals, each rounded to 256.
inline uint64_t scan_states_bytes(const nsfps_scan_args &a) {
  const uint64_t chunks = host_ceil_div(a.length, kChunk);
  return (4 * a.batch * a.heads * chunks * a.head_dim * a.state_dim + 255) & ~255ull;
}
inline uint64_t scan_totals_bytes(const nsfps_scan_args &a) {
  return (4 * a.batch * a.heads * host_ceil_div(a.length, kChunk) + 255) & ~255ull;
}

inline ScanDev scan_dev(const nsfps_scan_args &a) {
  ScanDev s = {};
  s.batch = (uint32_t)a.batch;
  s.length = (uint32_t)a.length;
  s.heads = a.heads;
  s.groups = a.groups;
  s.head_dim = a.head_dim;
  s.state_dim = a.state_dim;
  s.chunks = (uint32_t)host_ceil_div(a.length, kChunk);
  s.ptiles = (a.head_dim + kPTile - 1) / kPTile;
  s.x = a.x;
  s.b = a.b;
  s.c = a.c;
  s.dt = a.dt;
  s.y = a.y;
  s.a = a.d_a;
  s.d = a.d_d;
  s.dt_bias = a.d_dt_bias;
  s.lengths = a.d_lengths;
  s.positions = a.d_positions;
  s.slots = a.d_slots;
  s.state = a.d_state;
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2, v = 16 / size;
  s.wide_x = rows_wide(a.x, size) && a.head_dim % v == 0;
  s.wide_bc = rows_wide(a.b, size) && rows_wide(a.c, size) && a.state_dim % v == 0;
  s.wide_y = rows_wide(a.y, size) && a.head_dim % v == 0;
  return s;
}

// f(element type, state_dim rounded up to a template's)
template <typename F>
hipError_t scan_by_type(uint32_t dtype, uint32_t state_dim, F f) {
  const auto by_state = [&](auto t) {
    if (state_dim <= 32) return f(t, std::integral_constant<int, 32>());
    if (state_dim <= 64) return f(t, std::integral_constant<int, 64>());
    return f(t, std::integral_constant<int, 128>());
  };
  return dtype == NSFPS_F32 ? by_state(float()) : by_state(bf16());
}

}  // namespace seq
}  // namespace nsfps
