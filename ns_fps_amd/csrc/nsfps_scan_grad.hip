// Gradient of the selective state space scan.
//
// With a chunk of 64 tokens, H the state it starts from, dH the gradient of the
// state it ends with, s the running sum of delta a, S = c b^T, W = dy x^T (both
// 64 x 64), L_ij = exp(s_i - s_j) for j <= i and 0 above, M_ij = L_ij delta_j S_ij,
// G_ij = L_ij delta_j W_ij, w_j = delta_j exp(s_last - s_j), e_i = exp(s_i):
//   dx_j = sum_i M_ij dy_i + w_j dH b_j + d dy_j
//   db_j = sum_i G_ij c_i + w_j dH^T x_j         (added over a group's heads)
//   dc_i = sum_j G_ij b_j + e_i H^T dy_i         (the same)
// and, with T = M W elementwise (its diagonal may be left out), the exponent delta_t a of a token gets
//   da_t = sum_{i>=t} (sum_j T_ij + c_i . e_i H^T dy_i) - sum_{j>=t} sum_i T_ij
//          + sum_{j<t} w_j x_j . dH b_j + exp(s_last) <dH, H>,
// all terms from inside the chunk, so nothing cancels over the sequence.  Then
// ddelta_t = a da_t + (what came through delta_t itself), ddt = ddelta sigmoid(raw).
//
// H and dH come from the forward's chunk sums and pass, and from the same two
// kernels run over dy and c from the sequence's end (nothing is kept from the
// forward call); then every chunk is done by itself, one workgroup per chunk
// and group: a wave owns 16 tokens, as rows i for dc and as columns j for dx
// and db, finds S and W in both orientations so that the weighted tiles are
// operands as they lie in its registers, and goes through the group's heads
// with db and dc in registers: the sum over shared heads has a fixed order.
#include "nsfps_launch.h"
#include "nsfps_scan_device.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

struct GradDev {
  nsfps_rows dy, dx, db, dc, ddt;
  const float *ends;   // dH: [batch][heads][chunks][head_dim][state_dim]
  float *part;         // [3][heads][batch * chunks]: da, dd, ddt_bias
  uint32_t wide_dy, wide_dx, wide_dbc;
};

template <typename T, int NT>
struct GradLds {
  static constexpr int kTerms = Terms<T, 3>::kN;
  T x[kChunk * kLd<T, (int)kPTile>], dy[kChunk * kLd<T, (int)kPTile>];
  T b[kChunk * kLd<T, NT>], c[kChunk * kLd<T, NT>];
  T h[kTerms][kPTile * kLd<T, NT>];  // H, then dH
  Steps st;
  // by token: T's sums over j < i and (without delta_j) over i > j, its
  // diagonal (without delta), c_i . e_i H^T dy_i, x_j . dH b_j to the chunk's end
  double row_t[kChunk], col_u[kChunk];
  float diag[kChunk], from[kChunk], thru[kChunk];
  float red[8];  // per wave: <dH, H>, sum dy.x
};

// 64 x NT values of a state, head_dim rows from p0 on, as three terms each
// (float32: one).  With H given too, returns this thread's part of <v, H>.
template <typename T, int NT>
__device__ __forceinline__ float load_state(GradLds<T, NT> &m, const float *v, const float *with,
                                            uint32_t rows, uint32_t cols) {
  float dot = 0.f;
  for (uint32_t e = threadIdx.x; e < kPTile * (NT / 4); e += 256) {
    const uint32_t p = e / (NT / 4), n = (e % (NT / 4)) * 4;
    f32x4 q = {0.f, 0.f, 0.f, 0.f};
    if (p < rows)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (n + i < cols) {
          q[i] = v[p * cols + n + i];
          if (with) dot = fmaf(q[i], with[p * cols + n + i], dot);
        }
    const Terms<T, 3> t = split<T, 3>(q);
#pragma unroll
    for (int k = 0; k < Terms<T, 3>::kN; ++k)
      *(Quad<T> *)(m.h[k] + p * kLd<T, NT> + n) = t.q[k];
  }
  return dot;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// over the four quads of a column (lanes l, 16 + l, 32 + l, 48 + l)
template <typename V>
__device__ __forceinline__ V column_sum(V v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Four values of a lane's column to a row of global memory.
template <typename T>
__device__ __forceinline__ void store_quad(T *dst, f32x4 v, uint32_t at, uint32_t cols, bool wide) {
  if (wide) {
    const float o[4] = {v[0], v[1], v[2], v[3]};
    if (at < cols) store_f32<T, 4>(dst + at, o);
  } else {
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) {
      const float o[1] = {v[r]};
      if (at + r < cols) store_f32<T, 1>(dst + at + r, o);
    }
  }
}

template <typename T, int NT>
__global__ __launch_bounds__(256) void k_scan_grad(ScanDev s, GradDev gr, uint64_t work) {
  extern __shared__ __attribute__((aligned(16))) char s_raw[];
  GradLds<T, NT> &m = *(GradLds<T, NT> *)s_raw;
  constexpr int ldx = kLd<T, (int)kPTile>, ldn = kLd<T, NT>, kT3 = Terms<T, 3>::kN,
                kT2 = Terms<T, 2>::kN, kNt = NT / 16;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, l = lane & 15u;
  const uint32_t each = s.heads / s.groups;  // heads of a group
  const int own = 16 * wave + l;             // this lane's token, as i and as j
  for (uint64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const uint32_t grp = (uint32_t)(w % s.groups);
    const uint64_t bc = w / s.groups;
    const uint32_t c = (uint32_t)(bc % s.chunks), b = (uint32_t)(bc / s.chunks);
    const uint32_t len = scan_length(s, b), t0 = c * kChunk;
    const uint32_t out_rows = min(kChunk, s.length - t0);
    const uint32_t rows = t0 < len ? min(kChunk, len - t0) : 0u;
    const bool writes = (uint32_t)own < out_rows;
    const auto rows_at = [&](const nsfps_rows &r) {
      return (T *)r.p + (uint64_t)b * r.batch_stride + (uint64_t)t0 * r.row_stride;
    };
    T *const db_row = rows_at(gr.db) + (uint64_t)own * gr.db.row_stride + grp * s.state_dim;
    T *const dc_row = rows_at(gr.dc) + (uint64_t)own * gr.dc.row_stride + grp * s.state_dim;
    if (rows == 0) {  // past the sequence's end: zeros
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
      if (writes) {
        for (uint32_t nt = 0; nt < kNt; ++nt) {
          store_quad<T>(db_row, z, 16 * nt + 4 * g, s.state_dim, false);
          store_quad<T>(dc_row, z, 16 * nt + 4 * g, s.state_dim, false);
        }
        T *dx_row = rows_at(gr.dx) + (uint64_t)own * gr.dx.row_stride;
        T *ddt_row = rows_at(gr.ddt) + (uint64_t)own * gr.ddt.row_stride;
        for (uint32_t p = grp * each * s.head_dim + g; p < (grp + 1) * each * s.head_dim; p += 4)
          store_quad<T>(dx_row + p, z, 0, 1, false);
        for (uint32_t h = grp * each + g; h < (grp + 1) * each; h += 4)
          store_quad<T>(ddt_row + h, z, 0, 1, false);
      }
      if (threadIdx.x < 3)
        for (uint32_t h = grp * each; h < (grp + 1) * each; ++h)
          gr.part[((uint64_t)threadIdx.x * s.heads + h) * s.batch * s.chunks + bc] = 0.f;
      continue;
    }
    load_tile<T, NT>(m.b, rows_at(s.b) + grp * s.state_dim, s.b.row_stride, rows, s.state_dim,
                     s.wide_bc);
    load_tile<T, NT>(m.c, rows_at(s.c) + grp * s.state_dim, s.c.row_stride, rows, s.state_dim,
                     s.wide_bc);
    __syncthreads();

    // S with this wave's tokens as columns j (tiles of rows i >= its own) and,
    // transposed, as columns i (tiles of rows j <= its own)
    f32x4 s_j[4] = {}, s_i[4] = {};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int nt = 0; nt < kNt; nt += 2) {
        const int k0 = 16 * nt + 4 * g, k1 = k0 + 16;
        if (t >= (int)wave)
          mma_apart(s_j[t], quad_row<T>(m.c, ldn, 16 * t + l, k0), quad_row<T>(m.c, ldn, 16 * t + l, k1),
              quad_row<T>(m.b, ldn, own, k0), quad_row<T>(m.b, ldn, own, k1));
        if (t <= (int)wave)
          mma_apart(s_i[t], quad_row<T>(m.b, ldn, 16 * t + l, k0), quad_row<T>(m.b, ldn, 16 * t + l, k1),
              quad_row<T>(m.c, ldn, own, k0), quad_row<T>(m.c, ldn, own, k1));
      }
    }

    f32x4 db[kNt] = {}, dc[kNt] = {};
    for (uint32_t h = grp * each; h < (grp + 1) * each; ++h) {
      // ---- W in both orientations, over head_dim
      f32x4 w_j[4] = {}, w_i[4] = {};
      const auto load_xdy = [&](uint32_t p0) {
        load_tile<T, (int)kPTile>(m.x, rows_at(s.x) + h * s.head_dim + p0, s.x.row_stride, rows,
                                  s.head_dim - p0, s.wide_x);
        load_tile<T, (int)kPTile>(m.dy, rows_at(gr.dy) + h * s.head_dim + p0, gr.dy.row_stride,
                                  rows, s.head_dim - p0, gr.wide_dy);
      };
      for (uint32_t pt = 0; pt < s.ptiles; ++pt) {
        load_xdy(pt * kPTile);
        if (pt == 0 && wave == 0) chunk_steps<T>(s, m.st, b, h, t0, len);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int kt = 0; kt < (int)kPTile / 16; kt += 2) {
            const int k0 = 16 * kt + 4 * g, k1 = k0 + 16;
            if (t >= (int)wave)
              mma_apart(w_j[t], quad_row<T>(m.dy, ldx, 16 * t + l, k0),
                  quad_row<T>(m.dy, ldx, 16 * t + l, k1), quad_row<T>(m.x, ldx, own, k0),
                  quad_row<T>(m.x, ldx, own, k1));
            if (t <= (int)wave)
              mma_apart(w_i[t], quad_row<T>(m.x, ldx, 16 * t + l, k0),
                  quad_row<T>(m.x, ldx, 16 * t + l, k1), quad_row<T>(m.dy, ldx, own, k0),
                  quad_row<T>(m.dy, ldx, own, k1));
          }
        }
        if (s.ptiles > 1) __syncthreads();  // the tiles are loaded again
      }

      // ---- the weighted tiles: M and G as columns j, G as columns i; sums of T
      Terms<T, 2> m_j[4], g_j[4], g_i[4];
      // L_ij S_ij W_ij without the diagonal, which counts nowhere: sums over i
      // (u_off) and, times delta_j, over j (rt).  In float64, from products
      // rounded alike in both orientations: below, sums over rows are taken
      // from sums over columns, and what is in both must go.
      double u_off = 0.0, rt = 0.0;
      float diag = 0.f, dd = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 mj = {0.f, 0.f, 0.f, 0.f}, gj = mj, gi = mj;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int o = 16 * t + 4 * g + r;  // the tile's other token
          if (t >= (int)wave && o >= own) {
            const float lw = decay_between(m.st, o, own);
            const float ls = lw * s_j[t][r];
            mj[r] = ls * m.st.delta[own];
            gj[r] = lw * m.st.delta[own] * w_j[t][r];
            if (o == own) {
              dd = w_j[t][r];
              diag = ls * dd;
            } else {
              u_off += (double)(ls * w_j[t][r]);
            }
          }
          if (t <= (int)wave && o <= own) {
            const float lw = decay_between(m.st, own, o);
            gi[r] = lw * m.st.delta[o] * w_i[t][r];
            if (o != own) rt = fma((double)((lw * s_i[t][r]) * w_i[t][r]), (double)m.st.delta[o], rt);
          }
        }
        m_j[t] = split<T, 2>(mj);
        g_j[t] = split<T, 2>(gj);
        g_i[t] = split<T, 2>(gi);
      }
      u_off = column_sum(u_off);
      rt = column_sum(rt);
      diag = column_sum(diag);
      dd = wave_sum(dd);

      // ---- db and dc inside the chunk
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int k0 = 32 * tt + 4 * g, k1 = k0 + 16;
          if (2 * tt + 1 >= (int)wave) {
            const Quad<T> a0 = quad_col<T>(m.c, ldn, k0, 16 * nt + l);
            const Quad<T> a1 = quad_col<T>(m.c, ldn, k1, 16 * nt + l);
#pragma unroll
            for (int k = 0; k < kT2; ++k) mma(db[nt], a0, a1, g_j[2 * tt].q[k], g_j[2 * tt + 1].q[k]);
          }
          if (2 * tt <= (int)wave) {
            const Quad<T> a0 = quad_col<T>(m.b, ldn, k0, 16 * nt + l);
            const Quad<T> a1 = quad_col<T>(m.b, ldn, k1, 16 * nt + l);
#pragma unroll
            for (int k = 0; k < kT2; ++k) mma(dc[nt], a0, a1, g_i[2 * tt].q[k], g_i[2 * tt + 1].q[k]);
          }
        }
      }

      // ---- what passes through the states, 64 rows of them at a time
      const float e_i = exp2_fast(m.st.hi[own] + m.st.lo[own]);
      const float to_end = decay_between(m.st, kChunk - 1, own), w_end = m.st.delta[own] * to_end;
      float thru = 0.f, dot = 0.f;
      f32x4 dci[kNt] = {};
      for (uint32_t pt = 0; pt < s.ptiles; ++pt) {
        const uint32_t p0 = pt * kPTile, pn = min(kPTile, s.head_dim - p0);
        const uint64_t at = ((((uint64_t)b * s.heads + h) * s.chunks + c) * s.head_dim + p0) *
                            s.state_dim;
        if (s.ptiles > 1) load_xdy(p0);
        load_state<T, NT>(m, s.states + at, nullptr, pn, s.state_dim);
        __syncthreads();
        // H^T dy_i
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) {
          f32x4 low = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kt = 0; kt < (int)kPTile / 16; kt += 2) {
            const int k0 = 16 * kt + 4 * g, k1 = k0 + 16;
            const Quad<T> b0 = quad_row<T>(m.dy, ldx, own, k0), b1 = quad_row<T>(m.dy, ldx, own, k1);
#pragma unroll
            for (int k = kT3 - 1; k > 0; --k)
              mma(low, quad_col<T>(m.h[k], ldn, k0, 16 * nt + l),
                  quad_col<T>(m.h[k], ldn, k1, 16 * nt + l), b0, b1);
            mma_apart(dci[nt], quad_col<T>(m.h[0], ldn, k0, 16 * nt + l),
                      quad_col<T>(m.h[0], ldn, k1, 16 * nt + l), b0, b1);
          }
          dci[nt] += low;
        }
        __syncthreads();
        dot += load_state<T, NT>(m, gr.ends + at, s.states + at, pn, s.state_dim);
        __syncthreads();
        // dH^T x_j
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) {
          f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kt = 0; kt < (int)kPTile / 16; kt += 2) {
            const int k0 = 16 * kt + 4 * g, k1 = k0 + 16;
#pragma unroll
            for (int k = 0; k < kT3; ++k)
              mma(v, quad_col<T>(m.h[k], ldn, k0, 16 * nt + l),
                  quad_col<T>(m.h[k], ldn, k1, 16 * nt + l), quad_row<T>(m.x, ldx, own, k0),
                  quad_row<T>(m.x, ldx, own, k1));
          }
          db[nt] += v * w_end;
        }
        // dx: through the chunk, and dH b_j
        const float dskip = s.d ? s.d[h] : 0.f;
        T *const dx_row = rows_at(gr.dx) + (uint64_t)own * gr.dx.row_stride + h * s.head_dim + p0;
#pragma unroll
        for (int q = 0; q < (int)kPTile / 16; ++q) {
          f32x4 in = {0.f, 0.f, 0.f, 0.f}, thr = in, low = in;
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
            if (2 * tt + 1 >= (int)wave) {
              const Quad<T> a0 = quad_col<T>(m.dy, ldx, 32 * tt + 4 * g, 16 * q + l);
              const Quad<T> a1 = quad_col<T>(m.dy, ldx, 32 * tt + 16 + 4 * g, 16 * q + l);
#pragma unroll
              for (int k = 0; k < kT2; ++k) mma(in, a0, a1, m_j[2 * tt].q[k], m_j[2 * tt + 1].q[k]);
            }
#pragma unroll
          for (int nt = 0; nt < kNt; nt += 2) {
            const int k0 = 16 * nt + 4 * g, k1 = k0 + 16;
            const Quad<T> b0 = quad_row<T>(m.b, ldn, own, k0), b1 = quad_row<T>(m.b, ldn, own, k1);
#pragma unroll
            for (int k = kT3 - 1; k > 0; --k)
              mma(low, quad_row<T>(m.h[k], ldn, 16 * q + l, k0),
                  quad_row<T>(m.h[k], ldn, 16 * q + l, k1), b0, b1);
            mma_apart(thr, quad_row<T>(m.h[0], ldn, 16 * q + l, k0),
                      quad_row<T>(m.h[0], ldn, 16 * q + l, k1), b0, b1);
          }
          thr += low;
          const f32x4 xv = quad_f32(quad_row<T>(m.x, ldx, own, 16 * q + 4 * g));
          const f32x4 gv = quad_f32(quad_row<T>(m.dy, ldx, own, 16 * q + 4 * g));
          f32x4 o;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            thru = fmaf(xv[r], thr[r], thru);
            o[r] = (uint32_t)own < rows ? fmaf(dskip, gv[r], fmaf(w_end, thr[r], in[r])) : 0.f;
          }
          if (writes) store_quad<T>(dx_row, o, 16 * q + 4 * g, pn, gr.wide_dx);
        }
        if (pt + 1 < s.ptiles) __syncthreads();
      }
      thru = column_sum(thru) * to_end;  // per delta_j
      // dc through the states, and its part of the exponents' gradient
      float ri = 0.f;
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
        const f32x4 cv = quad_f32(quad_row<T>(m.c, ldn, own, 16 * nt + 4 * g));
#pragma unroll
        for (int r = 0; r < 4; ++r) ri = fmaf(cv[r], dci[nt][r], ri);
        dc[nt] += dci[nt] * e_i;
      }
      if (g == 0) {
        m.row_t[own] = rt;
        m.col_u[own] = u_off;
        m.thru[own] = thru;
      }
      ri = column_sum(ri) * e_i;
      if (g == 1) {
        m.from[own] = ri;
        m.diag[own] = diag;
      }
      dot = wave_sum(dot);
      if (lane == 0) {
        m.red[wave] = dot;
        m.red[4 + wave] = dd;
      }
      __syncthreads();
      // ---- the exponents: sums over the chunk's tokens from each on, and before it
      if (wave == 0) {
        const float delta = m.st.delta[lane];
        double after = m.row_t[lane] - (double)delta * m.col_u[lane];  // cancels, so first
        double from = m.from[lane];
        const double mine = (double)delta * m.thru[lane];
        double before = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const double a2 = __shfl_down(after, off, 64), b2 = __shfl_up(before, off, 64);
          const double f2 = __shfl_down(from, off, 64);
          if (lane + off < 64) after += a2, from += f2;
          if (lane >= (uint32_t)off) before += b2;
        }
        const float whole = exp2_fast(m.st.hi[kChunk - 1] + m.st.lo[kChunk - 1]) *
                            (m.red[0] + m.red[1] + m.red[2] + m.red[3]);
        const float da = (float)(after + from + (before - mine)) + whole;
        float ddt = 0.f;
        if (lane < rows)
          ddt = fmaf(s.a[h], da, (float)m.col_u[lane] + m.diag[lane] + m.thru[lane]) *
                sigmoid(raw_step<T>(s, b, h, t0 + lane));
        const float o[1] = {ddt};
        if (lane < out_rows)
          store_f32<T, 1>(rows_at(gr.ddt) + (uint64_t)lane * gr.ddt.row_stride + h, o);
        const float sda = wave_sum(delta * da), sdt = wave_sum(ddt);
        if (lane == 0) {
          const uint64_t per = (uint64_t)s.batch * s.chunks;
          gr.part[(uint64_t)h * per + bc] = sda;
          gr.part[((uint64_t)s.heads + h) * per + bc] = m.red[4] + m.red[5] + m.red[6] + m.red[7];
          gr.part[((uint64_t)2 * s.heads + h) * per + bc] = sdt;
        }
      }
      __syncthreads();
    }
    if (writes) {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
        store_quad<T>(db_row, db[nt], 16 * nt + 4 * g, s.state_dim, gr.wide_dbc);
        store_quad<T>(dc_row, dc[nt], 16 * nt + 4 * g, s.state_dim, gr.wide_dbc);
      }
    }
    __syncthreads();
  }
}

// One workgroup per head and parameter: the chunks' parts in a fixed order.
__global__ __launch_bounds__(256) void k_scan_grad_join(const float *__restrict__ part,
                                                        uint64_t count, uint32_t heads, float *da,
                                                        float *dd, float *ddt_bias) {
  __shared__ double s_sum[4];
  float *const out[3] = {da, dd, ddt_bias};
  const uint32_t h = blockIdx.x, k = blockIdx.y;
  const float *p = part + ((uint64_t)k * heads + h) * count;
  double sum = 0.0;
  for (uint64_t i = threadIdx.x; i < count; i += 256) sum += p[i];
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0 && out[k]) out[k][h] = (float)(s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]);
}

uint64_t part_bytes(const nsfps_scan_args &a) {
  return (12 * a.batch * a.heads * host_ceil_div(a.length, kChunk) + 255) & ~255ull;
}

}  // namespace

uint64_t scan_grad_bytes(const nsfps_scan_args &a) {
  return 2 * scan_states_bytes(a) + scan_totals_bytes(a) + part_bytes(a);
}

hipError_t launch_scan_grad(const nsfps_scan_args &a, const nsfps_scan_grads &g, hipStream_t st) {
  ScanDev s = scan_dev(a);
  char *const ws = (char *)a.workspace;
  s.states = (float *)ws;
  float *const ends = (float *)(ws + scan_states_bytes(a));
  s.totals = (float *)(ws + 2 * scan_states_bytes(a));
  GradDev d = {};
  d.dy = g.dy;
  d.dx = g.dx;
  d.db = g.db;
  d.dc = g.dc;
  d.ddt = g.ddt;
  d.ends = ends;
  d.part = (float *)(ws + 2 * scan_states_bytes(a) + scan_totals_bytes(a));
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2, v = 16 / size;
  d.wide_dy = rows_wide(g.dy, size) && a.head_dim % v == 0;
  d.wide_dx = rows_wide(g.dx, size) && a.head_dim % v == 0;
  d.wide_dbc = rows_wide(g.db, size) && rows_wide(g.dc, size) && a.state_dim % v == 0;
  const uint64_t parts = a.batch * s.chunks, sums = parts * s.heads * s.ptiles,
                 work = parts * s.groups;
  const uint64_t values = a.batch * s.heads * (uint64_t)s.head_dim * s.state_dim;
  const auto run = [&](auto t, auto n) {
    using T = decltype(t);
    constexpr int NT = decltype(n)::value;
    k_scan_sums<T, NT, false><<<scan_grid(sums), 256, 0, st>>>(s, s.x, s.b, s.wide_x, s.wide_bc,
                                                               s.states, sums);
    k_scan_sums<T, NT, true><<<scan_grid(sums), 256, 0, st>>>(s, d.dy, s.c, d.wide_dy, s.wide_bc,
                                                              ends, sums);
    const uint32_t pass = scan_grid(host_ceil_div(values, 256));
    k_scan_pass<false><<<pass, 256, 0, st>>>(s, s.states, values);
    k_scan_pass<true><<<pass, 256, 0, st>>>(s, ends, values);
    constexpr size_t lds = sizeof(GradLds<T, NT>);
    static_assert(lds <= 160 * 1024, "LDS");
    const hipError_t e = hipFuncSetAttribute((const void *)k_scan_grad<T, NT>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    k_scan_grad<T, NT><<<scan_grid(work), 256, lds, st>>>(s, d, work);
    return hipGetLastError();
  };
  if (work) {
    const hipError_t e = scan_by_type(a.dtype, a.state_dim, run);
    if (e != hipSuccess) return e;
  }
  k_scan_grad_join<<<dim3(a.heads, 3), 256, 0, st>>>(d.part, parts, a.heads, g.d_da, g.d_dd,
                                                     g.d_ddt_bias);
  return hipGetLastError();
}

hipError_t preload_scan_grad_kernels() {
  return func_attributes(k_scan_grad<bf16, 64>, k_scan_grad_join);
}

}  // namespace nsfps
