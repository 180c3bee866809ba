// Pieces shared by the selective scan and its gradient: the chunk's steps and
// decays, the chunks' states, and the launch parameters.
#pragma once

#include "nsfps_mfma.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

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
  uint32_t seg, segs;  // chunks of a segment, segments of the longest sequence
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
struct alignas(16) Steps {  // read four at a time
  float delta[kChunk], hi[kChunk], lo[kChunk];
  float e[kChunk];     // decay from the chunk's start through the token
  float end[kChunk];   // decay from the token to the chunk's end
  float sig[kChunk];   // the derivative of the step by its raw value
  float total;         // log2 of the whole chunk's decay
};

__device__ __forceinline__ f32x4 quad_of(const float (&v)[kChunk], int at) {
  return *(const f32x4 *)(v + at);
}

// The raw step of a token (before softplus and its bias).
template <typename T>
__device__ __forceinline__ Raw<T, 1> raw_step(const ScanDev &s, uint32_t b, uint32_t h, uint32_t t) {
  return load_raw<T, 1>((const T *)s.dt.p + (uint64_t)b * s.dt.batch_stride +
                        (uint64_t)t * s.dt.row_stride + h);
}
template <typename T>
__device__ __forceinline__ float number(const Raw<T, 1> &r) {
  float v[1];
  numbers<T, 1>(r, v);
  return v[0];
}

// One wave fills the steps of a chunk from its lanes' raw steps; lanes past
// the sequence's end have inside = false and a step of 0.
__device__ __forceinline__ void chunk_steps(Steps &o, float raw, bool inside, float a) {
  const uint32_t lane = threadIdx.x & 63u;
  float slope;
  const float step = softplus(raw, slope), delta = inside ? step : 0.f;
  // A decay of 2^-1024 is 0 beside any float32, so no token counts for less:
  // the chunk's sums stay within 2^16, where the pair resolves 2^-31 however
  // far a token has gone, and -infinity stays out.  NaN stays in.  Past the end
  // nothing is added, whatever a is.
  double sum = inside ? (double)delta * (double)a * 1.4426950408889634074 : 0.0;
  sum = sum < -1024.0 ? -1024.0 : sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double o2 = __shfl_up(sum, off, 64);
    if (lane >= (uint32_t)off) sum += o2;
  }
  const double last = __shfl(sum, 63, 64);
  o.delta[lane] = delta;
  o.sig[lane] = inside ? slope : 0.f;
  o.hi[lane] = (float)sum;
  o.lo[lane] = (float)(sum - (double)(float)sum);
  o.e[lane] = exp2_fast((float)sum);
  o.end[lane] = exp2_fast((float)(last - sum));
  if (lane == 63) o.total = (float)sum;
}

inline uint32_t scan_grid(uint64_t work, uint64_t most = 1u << 20) {
  return (uint32_t)(work < most ? work : most);
}

inline uint64_t round256(uint64_t n) { return (n + 255) & ~255ull; }

// Chunks of a segment: all of a sequence's while the sequences fill the chip,
// two workgroups on each of 256 CUs; else as few as do.  us a call with 256,
// 512 and 1,024 workgroups: 65,536 tokens of 8 heads 223, 159, 173; 64 x 4,096
// tokens of 8 heads with gradient 1,615, 1,615, 1,919.  Segments of at least
// 4, 2 and 1 chunks: 1,000 tokens of 8 heads 28.2, 21.1, 18.7; 3 x 1,001 tokens
// of 6 heads in float32 with gradient 180, 134, 131.  (The second case takes
// 1,450 in all now, by later steps.)
inline uint32_t segment_chunks(uint64_t sequences, uint64_t chunks) {
  constexpr uint64_t kFill = 512;
  const uint64_t segs = std::max<uint64_t>(1, kFill / std::max<uint64_t>(1, sequences));
  return (uint32_t)std::max<uint64_t>(1, host_ceil_div(chunks, segs));
}

// What a sweep over segments needs beside its result: states and totals.
inline uint64_t carry_states_bytes(const ScanDev &s) {
  return round256(4ull * s.batch * s.heads * s.segs * s.head_dim * s.state_dim);
}
inline uint64_t carry_bytes(const ScanDev &s) {
  return s.segs < 2 ? 0
                    : carry_states_bytes(s) + round256(4ull * s.batch * s.heads * s.segs);
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
  s.seg = segment_chunks(a.batch * a.heads * s.ptiles, s.chunks);
  s.segs = (s.chunks + s.seg - 1) / s.seg;
  return s;
}

// Whether 16-byte accesses fit everywhere: the tensors' rows and their heads'
// and groups' parts.
inline bool scan_wide(const nsfps_scan_args &a, std::initializer_list<const nsfps_rows *> rows) {
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2, v = 16 / size;
  bool ok = a.head_dim % v == 0 && a.state_dim % v == 0 && (uintptr_t)a.d_state % 16 == 0;
  for (const nsfps_rows *r : rows) ok = ok && rows_wide(*r, size);
  return ok;
}

// f(element type, state_dim rounded up to a template's, 16-byte accesses)
template <typename F>
hipError_t scan_by_type(uint32_t dtype, uint32_t state_dim, bool wide, F f) {
  const auto by_wide = [&](auto t, auto n) {
    return wide ? f(t, n, std::true_type()) : f(t, n, std::false_type());
  };
  const auto by_state = [&](auto t) {
    if (state_dim <= 32) return by_wide(t, std::integral_constant<int, 32>());
    if (state_dim <= 64) return by_wide(t, std::integral_constant<int, 64>());
    return by_wide(t, std::integral_constant<int, 128>());
  };
  return dtype == NSFPS_F32 ? by_state(float()) : by_state(bf16());
}

}  // namespace seq

// The states each chunk starts from (reversed: the gradients each chunk's end
// state gets, from u = dy and v = c), without outputs; ws: carry_bytes.
hipError_t launch_states(const nsfps_scan_args &a, const seq::ScanDev &s, const nsfps_rows &u,
                         const nsfps_rows &v, float *store, bool reversed, char *ws,
                         hipStream_t st);
}  // namespace nsfps
