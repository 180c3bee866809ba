// Selective state space scan over prompts, and the one-token step.
//
// state_t = exp(delta_t a) state_{t-1} + delta_t x_t b_t^T,  y_t = state_t c_t + d x_t
// per head (state: head_dim x state_dim).  Over a chunk of 64 tokens, with s the
// running sum of delta a, this is products:
//   y_i = sum_{j<=i} exp(s_i - s_j) delta_j (c_i . b_j) x_j + exp(s_i) state_in c_i + d x_i
//   state_out = exp(s_last) state_in + sum_j exp(s_last - s_j) delta_j x_j b_j^T
// so the work is on the matrix cores and the sequence is only walked from
// chunk to chunk (k_scan_sweep).
#include "nsfps_launch.h"
#include "nsfps_scan_device.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

// ---- the sweep over a sequence's chunks
//
// One workgroup walks a segment of a sequence's chunks with a head's state (64
// rows of it) in registers, wave w holding rows 16w .. 16w+15 as the sum tiles
// [n][p] that the state's own update
//   state = decay(chunk) state + sum over tokens of weight u v^T
// accumulates into.  Forward: u = x, v = b, weight = delta_j * decay from j to
// the chunk's end.  Reversed, for the gradient: u = dy, v = c, weight = decay
// from the chunk's start through i, from the last chunk to the first.  The
// weighted u is split into three bfloat16 terms: states are float32 and keep
// float32 accuracy.
//
// kOut: the chunk's outputs too (forward).  The four waves share the ten
// 16 x 16 tiles of c b^T that the causal order leaves, weigh them and leave
// them in LDS as rows of operands; then each wave has its 16 columns of y from
// them and x, and from its rows of the state, which in its registers already
// are an operand.  Scores and states enter there as two bfloat16 terms (16
// bits): the output's own rounding to 8 bits stays the only one that shows.
//
// Few sequences: segments run side by side, a first sweep over them finding
// what each adds to the state (ends), k_scan_carry turning that into the state
// each starts from (starts).
struct SweepDev {
  nsfps_rows u, v;
  float *starts;  // [batch][heads][segs][head_dim][state_dim], or null: from the cache, or zero
  float *ends;    // the same shape: the segment's state after its chunks, or null
  float *totals;  // [batch][heads][segs], with ends: log2 of the segment's decay
  float *store;   // [batch][heads][chunks][head_dim][state_dim]: the state each chunk finds, or null
};

constexpr int kStepAhead = 4;  // chunks whose steps are found together, one by each wave

template <typename T, int NT, bool kOut>
struct SweepLds {
  static constexpr int kTerms = kOut ? Terms<T, 2>::kN : 1;
  T u[kChunk * kLd<T, (int)kPTile>], v[kChunk * kLd<T, NT>];
  T c[kOut ? kChunk * kLd<T, NT> : 16];
  T m[kTerms][kOut ? kChunk * kLd<T, (int)kChunk> : 16];  // weighted scores, rows i
  Steps st[kStepAhead];
};

// XCD-aware order of work: workgroups are dealt to the 8 XCDs in turn, so that
// item w is given to the XCD whose L2 already holds its neighbours' b and c.
__device__ __forceinline__ uint32_t xcd_item(uint32_t id, uint32_t work) {
  const uint32_t per = (work + 7) / 8;
  return (id % 8) * per + id / 8;
}

// This lane's part of a state: row p, columns 16nt + 4g .. + 3.
template <int kNt, bool kWideRows, bool kStore>
__device__ __forceinline__ void state_io(float *state, f32x4 (&v)[kNt], uint32_t p, uint32_t rows,
                                         uint32_t cols, uint32_t g) {
  if (p >= rows) return;
  NSFPS_GLOBAL_SEQ float *row = (NSFPS_GLOBAL_SEQ float *)(state + (uint64_t)p * cols);
#pragma unroll
  for (int nt = 0; nt < kNt; ++nt) {
    const uint32_t at = 16 * nt + 4 * g;
    if constexpr (kWideRows) {
      if (at < cols) {
        if constexpr (kStore)
          *(NSFPS_GLOBAL_SEQ f32x4 *)(row + at) = v[nt];
        else
          v[nt] = *(const NSFPS_GLOBAL_SEQ f32x4 *)(row + at);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (at + r < cols) {
          if constexpr (kStore)
            row[at + r] = v[nt][r];
          else
            v[nt][r] = row[at + r];
        }
    }
  }
}

// Bound by the chain from chunk to chunk: loads to LDS, barriers and products of
// one chunk follow each other, and two workgroups a CU are all that hides them.
// 65,536 tokens, 8 heads, 64 x 128 states, bfloat16: 49 us for the segments'
// states and 115 with outputs (1.0 TB/s over both); 64 sequences of up to 4,096 tokens
// of 8 heads, 64 x 64: 268 us with outputs, 187 without.
// Two workgroups a CU where their LDS allows it (160 KB): the compiler may then
// use 256 registers.
template <typename T, int NT, bool kOut>
constexpr int kSweepGroups = sizeof(SweepLds<T, NT, kOut>) <= 80 * 1024 ? 2 : 1;

template <typename T, int NT, bool kOut, bool kRev, bool kWideRows>
__global__ __launch_bounds__(256, (kSweepGroups<T, NT, kOut>)) void k_scan_sweep(ScanDev s,
                                                                                 SweepDev d,
                                                                                 uint32_t work) {
  extern __shared__ __attribute__((aligned(16))) char s_raw[];
  SweepLds<T, NT, kOut> &m = *(SweepLds<T, NT, kOut> *)s_raw;
  constexpr int ldu = kLd<T, (int)kPTile>, ldn = kLd<T, NT>, ldm = kLd<T, (int)kChunk>,
                kNt = NT / 16, kT2 = Terms<T, 2>::kN, kT3 = Terms<T, 3>::kN;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
                 g = lane >> 4, l = lane & 15u;
  const uint32_t hps = s.heads * s.ptiles;
  if constexpr (kOut) {  // the tiles above the diagonal that a product of 32 terms takes along
    for (uint32_t e = threadIdx.x; e < SweepLds<T, NT, kOut>::kTerms * kChunk * ldm; e += 256)
      (&m.m[0][0])[e] = from_f32<T>(0.f);
  }
  const uint32_t w = xcd_item(blockIdx.x, work);
  if (w >= work) return;
  const uint32_t hp = w % hps, sg = w / hps % s.segs, b = w / hps / s.segs;
  const uint32_t h = hp / s.ptiles, p0 = (hp % s.ptiles) * kPTile, pn = s.head_dim - p0;
  const uint32_t grp = h / (s.heads / s.groups), sn = s.state_dim;
  const uint32_t len = scan_length(s, b), n = (len + kChunk - 1) / kChunk;
  const uint32_t first = sg * s.seg, last = min(first + s.seg, s.chunks);  // chunks
  const uint32_t mine = n > first ? min(n, last) - first : 0;              // with tokens in them
  const uint64_t bh = (uint64_t)b * s.heads + h, pn_all = (uint64_t)s.head_dim * sn;
  const uint32_t p = 16 * wave + l;  // this lane's row of the state
  const bool works = 16 * wave < pn;
  f32x4 st[kNt] = {};
  float *cache = nullptr;
  if (kOut && s.state) {
    const int32_t slot = s.slots ? s.slots[b] : (int32_t)b;
    if (slot >= 0)
      cache = s.state + ((uint64_t)slot * s.heads + h) * pn_all + (uint64_t)p0 * sn;
  }
  const uint64_t seg_at = (bh * s.segs + sg) * pn_all + (uint64_t)p0 * sn;
  if (d.starts)
    state_io<kNt, kWideRows, false>(d.starts + seg_at, st, p, pn, sn, g);
  else if (cache && s.positions && s.positions[b] > 0)
    state_io<kNt, kWideRows, false>(cache, st, p, pn, sn, g);

  const T *const ub = (const T *)d.u.p + (uint64_t)b * d.u.batch_stride + h * s.head_dim + p0;
  const T *const vb = (const T *)d.v.p + (uint64_t)b * d.v.batch_stride + grp * sn;
  const T *const cb = (const T *)s.c.p + (uint64_t)b * s.c.batch_stride + grp * sn;
  T *const yb = (T *)s.y.p + (uint64_t)b * s.y.batch_stride + h * s.head_dim + p0;
  const auto chunk_at = [&](uint32_t k) { return kRev ? first + mine - 1 - k : first + k; };
  Tile<T, (int)kPTile, kWideRows> tu;
  Tile<T, NT, kWideRows> tv, tc;
  const auto fetch = [&](uint32_t k) {
    const uint32_t t0 = chunk_at(k) * kChunk, rows = len - t0;
    tu.fetch(ub + t0 * d.u.row_stride, d.u.row_stride, rows, pn);
    tv.fetch(vb + t0 * d.v.row_stride, d.v.row_stride, rows, sn);
    if constexpr (kOut) tc.fetch(cb + t0 * s.c.row_stride, s.c.row_stride, rows, sn);
  };
  // the raw step of the chunk this wave finds the steps of, one group ahead
  const float a_h = s.a[h], skip = kOut && s.d ? s.d[h] : 0.f, dt_bias = s.dt_bias ? s.dt_bias[h] : 0.f;
  Raw<T, 1> raw = zero_raw<T, 1>();
  const auto fetch_raw = [&](uint32_t k) {  // the last token again past the end
    raw = raw_step<T>(s, b, h, min(chunk_at(min(k + wave, mine - 1)) * kChunk + lane, len - 1));
  };
  float total = 0.f;
  wait_loads();
  if (mine) {
    fetch(0);
    fetch_raw(0);
  }
  for (uint32_t k = 0; k < mine; ++k) {
    const uint32_t c = chunk_at(k);
    const Steps &sp = m.st[k % kStepAhead];
    __syncthreads();  // the tiles of the chunk before are done with
    tu.put(m.u);
    tv.put(m.v);
    if constexpr (kOut) tc.put(m.c);
    if (k % kStepAhead == 0) {
      if (k + wave < mine)
        chunk_steps(m.st[wave], number(raw) + dt_bias, chunk_at(k + wave) * kChunk + lane < len, a_h);
      fetch_raw(k + kStepAhead);
    }
    __syncthreads();
    if (k + 1 < mine) fetch(k + 1);
    if (d.store)
      state_io<kNt, kWideRows, true>(d.store + (bh * s.chunks + c) * pn_all + (uint64_t)p0 * sn,
                                     st, p, pn, sn, g);

    if constexpr (kOut) {
      // tiles (i, j) of the lower triangle: 3, 3, 2, 2 a wave
      const int from = wave < 2 ? 3 * (int)wave : 2 + 2 * (int)wave, upto = from + (wave < 2 ? 3 : 2);
      for (int t = from; t < upto; ++t) {
        const int it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
        f32x4 q = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < NT / 32; ++kb)
          mma(q, pair_row(m.v, ldn, 16 * jt + l, kb, g), pair_row(m.c, ldn, 16 * it + l, kb, g));
        const int i = 16 * it + l, j0 = 16 * jt + 4 * g;
        const f32x4 dj = quad_of(sp.delta, j0), hj = quad_of(sp.hi, j0), lj = quad_of(sp.lo, j0);
        const float hi = sp.hi[i], lo = sp.lo[i];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          q[r] *= dj[r] * exp2_fast((hi - hj[r]) + (lo - lj[r]));
#pragma unroll
        for (int r = 0; r < 4; ++r) q[r] = j0 + r <= i ? q[r] : 0.f;
        const Terms<T, 2> sc = split<T, 2>(q);
#pragma unroll
        for (int e = 0; e < kT2; ++e) put_quad(m.m[e], ldm, i, j0, sc.q[e]);
      }
      __syncthreads();
    }
    if (works) {
      // x transposed: rows p, terms j (operand A of y, and times the weights B of the update)
      Pair<T> uq[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) uq[kb] = pair_col(m.u, ldu, kb, 16 * wave, g, l);
      if constexpr (kOut) {
        f32x4 own[4] = {}, carried[4] = {};
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
          for (int kb = 0; kb <= it / 2; ++kb)
#pragma unroll
            for (int e = 0; e < kT2; ++e)
              mma(own[it], uq[kb], pair_row(m.m[e], ldm, 16 * it + l, kb, g));
#pragma unroll
        for (int kb = 0; kb < NT / 32; ++kb) {
          const Terms<T, 2> h0 = split<T, 2>(st[2 * kb]), h1 = split<T, 2>(st[2 * kb + 1]);
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const Pair<T> cq = pair_row(m.c, ldn, 16 * it + l, kb, g);
#pragma unroll
            for (int e = 0; e < kT2; ++e) mma(carried[it], Pair<T>{h0.q[e], h1.q[e]}, cq);
          }
        }
        const uint32_t t0 = c * kChunk, out_rows = s.length - t0, rows = len - t0;
        const uint32_t po = 16 * wave + 4 * g;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const uint32_t i = 16 * it + l;
          const f32x4 xv = quad_f32(quad_row(m.u, ldu, i, po));
          const float e = sp.e[i];
          float o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = fmaf(skip, xv[r], fmaf(e, carried[it][r], own[it][r]));
            o[r] = i < rows ? v : 0.f;
          }
          T *dst = yb + (t0 + i) * s.y.row_stride + po;
          if (i < out_rows) {
            if constexpr (kWideRows) {
              if (po < pn) store_f32<T, 4>(dst, o);
            } else {
#pragma unroll
              for (uint32_t r = 0; r < 4; ++r) {
                const float o1[1] = {o[r]};
                if (po + r < pn) store_f32<T, 1>(dst + r, o1);
              }
            }
          }
        }
      }
      // the state's update
      const float keep = exp2_fast(sp.total);
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) st[nt] *= keep;
      f32x4 low[kNt] = {};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int j = 32 * kb + 4 * g;
        f32x4 q0 = quad_f32(uq[kb].q0), q1 = quad_f32(uq[kb].q1);
        if constexpr (kRev) {
          q0 *= quad_of(sp.e, j);
          q1 *= quad_of(sp.e, j + 16);
        } else {
          q0 *= quad_of(sp.delta, j) * quad_of(sp.end, j);
          q1 *= quad_of(sp.delta, j + 16) * quad_of(sp.end, j + 16);
        }
        const Terms<T, 3> u0 = split<T, 3>(q0), u1 = split<T, 3>(q1);
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) {
          const Pair<T> vq = pair_col(m.v, ldn, kb, 16 * nt, g, l);
#pragma unroll
          for (int e = kT3 - 1; e > 0; --e) mma(low[nt], vq, Pair<T>{u0.q[e], u1.q[e]});
          mma_apart(st[nt], vq, Pair<T>{u0.q[0], u1.q[0]});
        }
      }
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) st[nt] += low[nt];
    }
    total += sp.total;
  }
  if (d.ends) {
    state_io<kNt, kWideRows, true>(d.ends + seg_at, st, p, pn, sn, g);
    if (threadIdx.x == 0 && p0 == 0) d.totals[bh * s.segs + sg] = total;
  }
  if (cache && mine && n <= last)  // the sequence's last chunk
    state_io<kNt, kWideRows, true>(cache, st, p, pn, sn, g);
  if constexpr (kOut) {  // rows past the sequence's end
    const uint32_t from = max(n, first) * kChunk, upto = min(last * kChunk, s.length);
    const float z[1] = {0.f};
    const uint32_t cols = min(pn, kPTile);
    for (uint64_t e = threadIdx.x; from < upto && e < (uint64_t)(upto - from) * kPTile; e += 256)
      if (e % kPTile < cols)
        store_f32<T, 1>(yb + (from + e / kPTile) * s.y.row_stride + e % kPTile, z);
  }
}

// What each segment adds becomes the state each starts from (reversed: the
// gradient each ends with), in place; one thread per state value walks the
// sequence's segments, kRun of them loaded ahead.  64 segments of 8 heads of
// 64 x 128 states: 13 us, the walk's latency.
template <bool kRev>
__global__ __launch_bounds__(256) void k_scan_carry(ScanDev s, float *__restrict__ states,
                                                    const float *__restrict__ totals,
                                                    uint64_t values) {
  constexpr uint32_t kRun = 8;
  const uint32_t pn = s.head_dim * s.state_dim, n = s.segs;
  for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < values;
       e += (uint64_t)gridDim.x * 256) {
    const uint64_t bh = e / pn;
    const uint32_t b = (uint32_t)(bh / s.heads), at = (uint32_t)(e % pn);
    float run = 0.f;
    if (!kRev && s.state && s.positions && s.positions[b] > 0) {
      const int32_t slot = s.slots ? s.slots[b] : (int32_t)b;
      if (slot >= 0) run = s.state[((uint64_t)slot * s.heads + bh % s.heads) * pn + at];
    }
    float *st = states + bh * n * pn + at;
    const float *tot = totals + bh * n;
    for (uint32_t c0 = 0; c0 < n; c0 += kRun) {
      float v[kRun], t[kRun];
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) {
        const uint32_t i = min(c0 + k, n - 1), c = kRev ? n - 1 - i : i;
        v[k] = st[(uint64_t)c * pn];
        t[k] = tot[c];
      }
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) {
        if (c0 + k >= n) break;
        const uint32_t c = kRev ? n - 1 - (c0 + k) : c0 + k;
        st[(uint64_t)c * pn] = run;
        run = fmaf(exp2_fast(t[k]), run, v[k]);
      }
    }
  }
}

template <typename T, int NT, bool kOut, bool kRev, bool kWideRows>
hipError_t launch_sweep(const ScanDev &s, const SweepDev &d, hipStream_t st) {
  constexpr size_t lds = sizeof(SweepLds<T, NT, kOut>);
  static_assert(lds <= 160 * 1024, "LDS");
  const hipError_t e = hipFuncSetAttribute((const void *)k_scan_sweep<T, NT, kOut, kRev, kWideRows>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return e;
  // at most 2^22: sequences are split only while they are few
  const uint32_t work = s.batch * s.segs * s.heads * s.ptiles;
  k_scan_sweep<T, NT, kOut, kRev, kWideRows><<<(work + 7) / 8 * 8, 256, lds, st>>>(s, d, work);
  return hipGetLastError();
}

// The whole sweep: over segments first where there are several.  ws: carry_bytes.
template <typename T, int NT, bool kOut, bool kRev, bool kWideRows>
hipError_t run_sweep(const ScanDev &s, SweepDev d, char *ws, hipStream_t st) {
  if (s.segs > 1) {
    SweepDev first = d;
    first.store = nullptr;
    first.ends = (float *)ws;
    first.totals = (float *)(ws + carry_states_bytes(s));
    hipError_t e = launch_sweep<T, NT, false, kRev, kWideRows>(s, first, st);
    if (e != hipSuccess) return e;
    const uint64_t values = (uint64_t)s.batch * s.heads * s.head_dim * s.state_dim;
    k_scan_carry<kRev><<<scan_grid(host_ceil_div(values, 256)), 256, 0, st>>>(
        s, first.ends, first.totals, values);
    d.starts = first.ends;
  }
  return launch_sweep<T, NT, kOut, kRev, kWideRows>(s, d, st);
}

// ---- one token

// One token of a request and head: 256 threads, 16 rows of the state at a
// time, 16 threads a row, kSets times.  The state is all the traffic that
// counts: its loads go out first and wait while the workgroup convolves the
// channels it needs itself (its rows' x; b and c of its group).  The ring
// holds `width` entries, of which the convolution reads the last width - 1 and
// this token's replaces the oldest, so a workgroup that writes its entry
// disturbs no other that still reads.  512 requests of 16 heads of 64 x 128
// states: 105 us, 5.2 TB/s of the 546 MB (an update of 4 GiB in place reaches
// 5.9); one request of 8 heads: 5 us, one chain of loads.
//
// kV: 4 state values a load where state_dim and the cache allow it, kCols of
// those a thread.  kSets: 4 (a head of 64 rows) where that still gives every CU
// a workgroup, else 1: few requests need the width of the chip more than they
// need the convolution done once.  us with 1 and with 4, 64 x 128 states,
// bfloat16: 128 heads of all requests 5.0, 6.2; 256 6.7, 6.8; 512 9.8, 8.3;
// 1,024 17.7, 13.1; 64 x 64 states: 128 4.1, 4.5; 256 5.3, 4.8; 512 7.7, 5.6;
// 1,024 12.1, 7.6.
template <typename T, int W, int kV, int kCols, int kSets>
__global__ __launch_bounds__(256) void k_scan_step(nsfps_step_args a, uint32_t ptiles) {
  constexpr uint32_t kRows = 16 * kSets;
  __shared__ float s_bc[2][128 + 4], s_x[kRows];
  const uint32_t pt = blockIdx.x % ptiles, h = (blockIdx.x / ptiles) % a.heads;
  const uint64_t b = blockIdx.x / ptiles / a.heads;
  const uint32_t p0 = pt * kRows, rows = min(kRows, a.head_dim - p0), n = a.state_dim;
  const uint32_t grp = h / (a.heads / a.groups);
  const uint64_t hp = (uint64_t)a.heads * a.head_dim, gn = (uint64_t)a.groups * n,
                 channels = hp + 2 * gn;
  T *const y = (T *)a.d_y + b * a.y_stride + (uint64_t)h * a.head_dim + p0;
  const int32_t slot = a.d_slots ? a.d_slots[b] : (int32_t)b;
  if (slot < 0) {
    const float z[1] = {0.f};
    if (threadIdx.x < rows) store_f32<T, 1>(y + threadIdx.x, z);
    return;
  }
  const uint32_t pos = a.d_positions[b] > 0 ? (uint32_t)a.d_positions[b] : 0u;
  const uint32_t r = threadIdx.x / 16, l = threadIdx.x % 16;
  float *const state = a.d_state + (((uint64_t)slot * a.heads + h) * a.head_dim + p0) * n;
  float st[kSets][kCols][kV];
#pragma unroll
  for (int q = 0; q < kSets; ++q)
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const uint32_t p = 16 * q + r, k = kV * (l + 16 * c);
#pragma unroll
      for (int i = 0; i < kV; ++i) st[q][c][i] = 0.f;
      if (pos && p < rows && k < n) load_f32<float, kV>(state + p * n + k, st[q][c]);
    }
  const T *xbc = (const T *)a.d_xbc + b * a.xbc_stride, *weight = (const T *)a.d_weight;
  T *const ring = (T *)a.d_cache + (uint64_t)slot * W * channels;
  float raw[1];
  load_f32<T, 1>((const T *)a.d_dt + b * a.dt_stride + h, raw);
  const float a_h = a.d_a[h], skip = a.d_d ? a.d_d[h] : 0.f;
  if (a.d_dt_bias) raw[0] += a.d_dt_bias[h];
  uint32_t entry[W];  // the ring's entries, this token's and those before it
#pragma unroll
  for (int back = 0; back < W; ++back) entry[back] = (pos + W - back) % W;
  // channels: rows of x, then n of b, then n of c
  for (uint32_t e = threadIdx.x; e < rows + 2 * n; e += 256) {
    const bool is_x = e < rows;
    const uint32_t o = is_x ? e : e - rows, k = !is_x && o >= n;  // 0: b, 1: c
    const uint64_t ch = is_x ? (uint64_t)h * a.head_dim + p0 + o
                             : hp + k * gn + (uint64_t)grp * n + (o - k * n);
    float in[W][1], w[W][1], pre[1] = {0.f};
    if (a.d_bias) load_f32<T, 1>((const T *)a.d_bias + ch, pre);
    load_f32<T, 1>(xbc + ch, in[0]);
#pragma unroll
    for (int back = 0; back < W; ++back) {
      load_f32<T, 1>(weight + ch * W + (W - 1 - back), w[back]);
      if (back) {
        in[back][0] = 0.f;
        if (pos >= (uint32_t)back) load_f32<T, 1>(ring + entry[back] * channels + ch, in[back]);
      }
    }
#pragma unroll
    for (int back = W - 1; back >= 0; --back) pre[0] = fmaf(w[back][0], in[back][0], pre[0]);
    const float v = pre[0] * sigmoid(pre[0]);
    if (is_x)
      s_x[o] = v;
    else
      s_bc[k][o - k * n] = v;
    // one workgroup owns each channel's ring entry
    if (is_x || (pt == 0 && h % (a.heads / a.groups) == 0))
      store_f32<T, 1>(ring + entry[0] * channels + ch, in[0]);
  }
  float slope;
  const float delta = softplus(raw[0], slope), log_decay = delta * a_h;
  // with the bits that the product's rounding took (past -200 it may be infinite)
  const float decay =
      exp_f32(log_decay, log_decay < -200.f ? 0.f : fmaf(delta, a_h, -log_decay));
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kSets; ++q) {
    const uint32_t p = 16 * q + r;
    float sum = 0.f;
    if (p < rows) {
      const float xd = delta * s_x[p];
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const uint32_t k = kV * (l + 16 * c);
        if (k >= n) continue;
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          st[q][c][i] = fmaf(xd, s_bc[0][k + i], decay * st[q][c][i]);
          sum = fmaf(st[q][c][i], s_bc[1][k + i], sum);
        }
        store_f32<float, kV>(state + p * n + k, st[q][c]);
      }
    }
#pragma unroll
    for (int off = 8; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (p < rows && l == 0) {
      const float o[1] = {fmaf(skip, s_x[p], sum)};
      store_f32<T, 1>(y + p, o);
    }
  }
}

}  // namespace

// Never 0, though a call of many sequences needs none: what a caller has to
// bring does not hang on how the work is split.
uint64_t scan_bytes(const nsfps_scan_args &a) {
  return std::max<uint64_t>(256, carry_bytes(scan_dev(a)));
}

hipError_t launch_scan(const nsfps_scan_args &a, hipStream_t st) {
  const ScanDev s = scan_dev(a);
  SweepDev d = {};
  d.u = s.x;
  d.v = s.b;
  const bool wide = scan_wide(a, {&a.x, &a.b, &a.c, &a.y});
  return scan_by_type(a.dtype, a.state_dim, wide, [&](auto t, auto n, auto w) {
    return run_sweep<decltype(t), decltype(n)::value, true, false, decltype(w)::value>(
        s, d, (char *)a.workspace, st);
  });
}

hipError_t launch_states(const nsfps_scan_args &a, const ScanDev &s, const nsfps_rows &u,
                         const nsfps_rows &v, float *store, bool reversed, char *ws,
                         hipStream_t st) {
  SweepDev d = {};
  d.u = u;
  d.v = v;
  d.store = store;
  return scan_by_type(a.dtype, a.state_dim, scan_wide(a, {&u, &v}), [&](auto t, auto n, auto w) {
    using T = decltype(t);
    constexpr int NT = decltype(n)::value;
    constexpr bool kWideRows = decltype(w)::value;
    return reversed ? run_sweep<T, NT, false, true, kWideRows>(s, d, ws, st)
                    : run_sweep<T, NT, false, false, kWideRows>(s, d, ws, st);
  });
}

hipError_t launch_scan_step(const nsfps_step_args &a, hipStream_t st) {
  const bool many = a.batch * a.heads * host_ceil_div(a.head_dim, 64) >= 256;
  const uint32_t rows = many ? 64 : 16, ptiles = (a.head_dim + rows - 1) / rows;
  const uint32_t grid = (uint32_t)(a.batch * a.heads * ptiles);
  const bool wide = a.state_dim % 4 == 0 && (uintptr_t)a.d_state % 16 == 0;
  const auto go = [&](auto t, auto w, auto v, auto cols) {
    using T = decltype(t);
    constexpr int W = decltype(w)::value, V = decltype(v)::value, C = decltype(cols)::value;
    if (many)
      k_scan_step<T, W, V, C, 4><<<grid, 256, 0, st>>>(a, ptiles);
    else
      k_scan_step<T, W, V, C, 1><<<grid, 256, 0, st>>>(a, ptiles);
    return hipGetLastError();
  };
  const auto by_state = [&](auto t, auto w) {  // 16 threads a row, so 16 * V * C values
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 8> eight;
    if (wide) return a.state_dim <= 64 ? go(t, w, four, one) : go(t, w, four, two);
    return a.state_dim <= 64 ? go(t, w, one, four) : go(t, w, one, eight);
  };
  const auto by_width = [&](auto t) {
    switch (a.width) {
      case 2: return by_state(t, std::integral_constant<int, 2>());
      case 3: return by_state(t, std::integral_constant<int, 3>());
      default: return by_state(t, std::integral_constant<int, 4>());
    }
  };
  return a.dtype == NSFPS_F32 ? by_width(float()) : by_width(bf16());
}

hipError_t preload_scan_kernels() {
  return func_attributes(k_scan_sweep<bf16, 64, true, false, true>, k_scan_step<bf16, 4, 4, 2, 4>,
                         k_scan_carry<false>);
}

}  // namespace nsfps
