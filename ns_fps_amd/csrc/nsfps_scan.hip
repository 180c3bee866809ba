// Selective state space scan over prompts, and the one-token step.
//
// state_t = exp(delta_t a) state_{t-1} + delta_t x_t b_t^T,  y_t = state_t c_t + d x_t
// per head (state: head_dim x state_dim).  Over a chunk of 64 tokens, with s the
// running sum of delta a, this is products:
//   y_i = sum_{j<=i} exp(s_i - s_j) delta_j (c_i . b_j) x_j + exp(s_i) state_in c_i + d x_i
//   state_out = exp(s_last) state_in + sum_j exp(s_last - s_j) delta_j x_j b_j^T
// so the work is on the matrix cores and the sequence is only walked from
// chunk to chunk: the chunks' own sums are found side by side (k_scan_sums),
// a pass over them gives the state each chunk starts from (k_scan_pass), and
// the outputs are found side by side again (k_scan_out).
#include "nsfps_launch.h"
#include "nsfps_scan_device.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

// LDS of k_scan_out, in elements of T
template <typename T, int NT>
struct OutLds {
  static constexpr int kTerms = Terms<T, 2>::kN;
  T x[kChunk * kLd<T, (int)kPTile>];
  T b[kChunk * kLd<T, NT>], c[kChunk * kLd<T, NT>];
  T h[kTerms][kPTile * kLd<T, NT>];
  Steps st;
};

// The outputs of a chunk, one wave per 16 tokens.  A wave finds its rows of
// c.b^T transposed, so that the weighted scores are, in its registers, the
// operand of the product with x.  Scores and states enter as two bfloat16
// terms (16 bits): the output's own rounding to 8 bits stays the only one
// that shows.
template <typename T, int NT>
__global__ __launch_bounds__(256) void k_scan_out(ScanDev s, uint64_t work) {
  extern __shared__ __attribute__((aligned(16))) char s_raw[];
  OutLds<T, NT> &m = *(OutLds<T, NT> *)s_raw;
  constexpr int ldx = kLd<T, (int)kPTile>, ldn = kLd<T, NT>, kTerms = OutLds<T, NT>::kTerms;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, l = lane & 15u;
  for (uint64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const uint32_t hp = (uint32_t)(w % (s.heads * s.ptiles));
    const uint64_t bc = w / (s.heads * s.ptiles);
    const uint32_t h = hp / s.ptiles, p0 = (hp % s.ptiles) * kPTile;
    const uint32_t c = (uint32_t)(bc % s.chunks), b = (uint32_t)(bc / s.chunks);
    const uint32_t len = scan_length(s, b), t0 = c * kChunk, pn = s.head_dim - p0;
    T *yr = (T *)s.y.p + (uint64_t)b * s.y.batch_stride + (uint64_t)t0 * s.y.row_stride +
            h * s.head_dim + p0;
    const uint32_t out_rows = min(kChunk, s.length - t0);
    if (t0 >= len) {  // past the sequence's end
      for (uint32_t e = threadIdx.x; e < kChunk * kPTile; e += 256) {
        const float z[1] = {0.f};
        if (e / kPTile < out_rows && e % kPTile < pn)
          store_f32<T, 1>(yr + (uint64_t)(e / kPTile) * s.y.row_stride + e % kPTile, z);
      }
      continue;
    }
    const uint32_t rows = min(kChunk, len - t0), grp = h / (s.heads / s.groups);
    load_tile<T, (int)kPTile>(m.x, (const T *)s.x.p + (uint64_t)b * s.x.batch_stride +
                                       (uint64_t)t0 * s.x.row_stride + h * s.head_dim + p0,
                              s.x.row_stride, rows, pn, s.wide_x);
    load_tile<T, NT>(m.b, (const T *)s.b.p + (uint64_t)b * s.b.batch_stride +
                              (uint64_t)t0 * s.b.row_stride + grp * s.state_dim,
                     s.b.row_stride, rows, s.state_dim, s.wide_bc);
    load_tile<T, NT>(m.c, (const T *)s.c.p + (uint64_t)b * s.c.batch_stride +
                              (uint64_t)t0 * s.c.row_stride + grp * s.state_dim,
                     s.c.row_stride, rows, s.state_dim, s.wide_bc);
    if (wave == 0) chunk_steps<T>(s, m.st, b, h, t0, len);
    const float *st = s.states +
                      (((uint64_t)b * s.heads + h) * s.chunks + c) * s.head_dim * s.state_dim +
                      (uint64_t)p0 * s.state_dim;
    for (uint32_t e = threadIdx.x; e < kPTile * (NT / 4); e += 256) {
      const uint32_t p = e / (NT / 4), n = (e % (NT / 4)) * 4;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (p < pn)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (n + i < s.state_dim) v[i] = st[p * s.state_dim + n + i];
      const Terms<T, 2> t = split<T, 2>(v);
#pragma unroll
      for (int k = 0; k < kTerms; ++k) *(Quad<T> *)(m.h[k] + p * ldn + n) = t.q[k];
    }
    __syncthreads();

    const int i = 16 * wave + l;  // this lane's token
    f32x4 from[kPTile / 16] = {}, own[kPTile / 16] = {};
    Quad<T> cq[NT / 16];
#pragma unroll
    for (int nt = 0; nt < NT / 16; ++nt) cq[nt] = quad_row<T>(m.c, ldn, i, 16 * nt + 4 * g);
    // state_in c_i
#pragma unroll
    for (int pt = 0; pt < (int)kPTile / 16; ++pt)
#pragma unroll
      for (int k = 0; k < kTerms; ++k)
#pragma unroll
        for (int nt = 0; nt < NT / 16; nt += 2)
          mma(from[pt], quad_row<T>(m.h[k], ldn, 16 * pt + l, 16 * nt + 4 * g),
              quad_row<T>(m.h[k], ldn, 16 * pt + l, 16 * nt + 16 + 4 * g), cq[nt], cq[nt + 1]);
    // the chunk's own tokens, 32 at a time
    for (uint32_t jj = 0; jj <= wave / 2; ++jj) {
      Terms<T, 2> sc[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int jt = 2 * jj + half;
        f32x4 q = {0.f, 0.f, 0.f, 0.f};
        if (jt <= (int)wave) {
#pragma unroll
          for (int nt = 0; nt < NT / 16; nt += 2)
            mma(q, quad_row<T>(m.b, ldn, 16 * jt + l, 16 * nt + 4 * g),
                quad_row<T>(m.b, ldn, 16 * jt + l, 16 * nt + 16 + 4 * g), cq[nt], cq[nt + 1]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * jt + 4 * g + r;
            q[r] = j <= i ? q[r] * m.st.delta[j] * decay_between(m.st, i, j) : 0.f;
          }
        }
        sc[half] = split<T, 2>(q);
      }
#pragma unroll
      for (int pt = 0; pt < (int)kPTile / 16; ++pt) {
        const Quad<T> a0 = quad_col<T>(m.x, ldx, 32 * jj + 4 * g, 16 * pt + l);
        const Quad<T> a1 = quad_col<T>(m.x, ldx, 32 * jj + 16 + 4 * g, 16 * pt + l);
#pragma unroll
        for (int k = 0; k < kTerms; ++k) mma(own[pt], a0, a1, sc[0].q[k], sc[1].q[k]);
      }
    }
    const float ei = exp2_fast(m.st.hi[i] + m.st.lo[i]), dh = s.d ? s.d[h] : 0.f;
    if ((uint32_t)i < out_rows) {
#pragma unroll
      for (int pt = 0; pt < (int)kPTile / 16; ++pt) {
        const int p = 16 * pt + 4 * g;
        const f32x4 xv = quad_f32(quad_row<T>(m.x, ldx, i, p));
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o[r] = t0 + i < len ? fmaf(dh, xv[r], fmaf(ei, from[pt][r], own[pt][r])) : 0.f;
        T *dst = yr + (uint64_t)i * s.y.row_stride + p;
        if (s.wide_y) {
          if ((uint32_t)p < pn) store_f32<T, 4>(dst, o);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float o1[1] = {o[r]};
            if ((uint32_t)(p + r) < pn) store_f32<T, 1>(dst + r, o1);
          }
        }
      }
    }
    __syncthreads();
  }
}

// ---- one token

constexpr uint32_t kStepRows = 16;  // state rows (head_dim) of a workgroup

// One token of a request and head: 256 threads, kStepRows rows of the state,
// 16 threads a row.  The workgroup convolves the channels it needs itself (its
// rows' x; b and c of its group): the ring holds `width` entries, of which the
// convolution reads the last width - 1 and this token's replaces the oldest,
// so a workgroup that writes its entry disturbs no other that still reads.
template <typename T, int W>
__global__ __launch_bounds__(256) void k_scan_step(nsfps_step_args a, uint32_t ptiles) {
  __shared__ float s_bc[2][128], s_x[kStepRows];
  const uint32_t pt = blockIdx.x % ptiles, h = (blockIdx.x / ptiles) % a.heads;
  const uint64_t b = blockIdx.x / ptiles / a.heads;
  const uint32_t p0 = pt * kStepRows, rows = min(kStepRows, a.head_dim - p0), n = a.state_dim;
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
  const T *xbc = (const T *)a.d_xbc + b * a.xbc_stride, *weight = (const T *)a.d_weight;
  T *const ring = (T *)a.d_cache + (uint64_t)slot * W * channels;
  // channels: rows of x, then n of b, then n of c
  for (uint32_t e = threadIdx.x; e < rows + 2 * n; e += 256) {
    const bool is_x = e < rows;
    const uint32_t k = is_x ? 0 : (e - rows) / n;  // 0: b, 1: c
    const uint64_t ch = is_x ? (uint64_t)h * a.head_dim + p0 + e
                             : hp + k * gn + (uint64_t)grp * n + (e - rows) % n;
    float in[1], w[1], pre[1] = {0.f};
    if (a.d_bias) load_f32<T, 1>((const T *)a.d_bias + ch, pre);
    load_f32<T, 1>(xbc + ch, in);
#pragma unroll
    for (int back = 1; back < W; ++back) {
      if (pos < (uint32_t)back) continue;
      float old[1];
      load_f32<T, 1>(ring + (uint64_t)((pos - back) % W) * channels + ch, old);
      load_f32<T, 1>(weight + ch * W + (W - 1 - back), w);
      pre[0] = fmaf(w[0], old[0], pre[0]);
    }
    load_f32<T, 1>(weight + ch * W + (W - 1), w);
    pre[0] = fmaf(w[0], in[0], pre[0]);
    const float v = pre[0] * sigmoid(pre[0]);
    if (is_x)
      s_x[e] = v;
    else
      s_bc[k][(e - rows) % n] = v;
    // one workgroup owns each channel's ring entry
    if (is_x || (pt == 0 && h % (a.heads / a.groups) == 0))
      store_f32<T, 1>(ring + (uint64_t)(pos % W) * channels + ch, in);
  }
  float raw[1];
  load_f32<T, 1>((const T *)a.d_dt + b * a.dt_stride + h, raw);
  const float delta = softplus(raw[0] + (a.d_dt_bias ? a.d_dt_bias[h] : 0.f));
  const float decay = exp2_fast(delta * a.d_a[h] * kLog2e);
  __syncthreads();
  const uint32_t r = threadIdx.x / 16, l = threadIdx.x % 16;
  float sum = 0.f;
  if (r < rows) {
    float *st = a.d_state + (((uint64_t)slot * a.heads + h) * a.head_dim + p0 + r) * n;
    const float xd = delta * s_x[r];
    for (uint32_t k = l; k < n; k += 16) {
      const float v = fmaf(xd, s_bc[0][k], pos ? decay * st[k] : 0.f);
      st[k] = v;
      sum = fmaf(v, s_bc[1][k], sum);
    }
  }
#pragma unroll
  for (int off = 8; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (r < rows && l == 0) {
    const float o[1] = {fmaf(a.d_d ? a.d_d[h] : 0.f, s_x[r], sum)};
    store_f32<T, 1>(y + r, o);
  }
}

}  // namespace

uint64_t scan_bytes(const nsfps_scan_args &a) {
  return scan_states_bytes(a) + scan_totals_bytes(a);
}

hipError_t launch_scan(const nsfps_scan_args &a, hipStream_t st) {
  ScanDev s = scan_dev(a);
  s.states = (float *)a.workspace;
  s.totals = (float *)((char *)a.workspace + scan_states_bytes(a));
  const uint64_t work = a.batch * s.chunks * s.heads * s.ptiles;
  const uint64_t values = a.batch * s.heads * (uint64_t)s.head_dim * s.state_dim;
  return scan_by_type(a.dtype, a.state_dim, [&](auto t, auto n) {
    using T = decltype(t);
    constexpr int NT = decltype(n)::value;
    k_scan_sums<T, NT, false><<<scan_grid(work), 256, 0, st>>>(s, s.x, s.b, s.wide_x, s.wide_bc,
                                                               s.states, work);
    k_scan_pass<false><<<scan_grid(host_ceil_div(values, 256)), 256, 0, st>>>(s, s.states, values);
    constexpr size_t lds = sizeof(OutLds<T, NT>);
    const hipError_t e = hipFuncSetAttribute((const void *)k_scan_out<T, NT>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    k_scan_out<T, NT><<<scan_grid(work), 256, lds, st>>>(s, work);
    return hipGetLastError();
  });
}

hipError_t launch_scan_step(const nsfps_step_args &a, hipStream_t st) {
  const uint32_t ptiles = (a.head_dim + kStepRows - 1) / kStepRows;
  const uint32_t grid = (uint32_t)(a.batch * a.heads * ptiles);
  const auto by_width = [&](auto t) {
    using T = decltype(t);
    switch (a.width) {
      case 2: k_scan_step<T, 2><<<grid, 256, 0, st>>>(a, ptiles); break;
      case 3: k_scan_step<T, 3><<<grid, 256, 0, st>>>(a, ptiles); break;
      default: k_scan_step<T, 4><<<grid, 256, 0, st>>>(a, ptiles);
    }
    return hipGetLastError();
  };
  return a.dtype == NSFPS_F32 ? by_width(float()) : by_width(bf16());
}

hipError_t preload_scan_kernels() {
  return func_attributes(k_scan_out<bf16, 64>, k_scan_step<bf16, 4>, k_scan_pass<false>);
}

}  // namespace nsfps
