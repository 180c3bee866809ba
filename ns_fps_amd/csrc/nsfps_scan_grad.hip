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
// In bfloat16 calls, what ends in a bfloat16 output alone (M, G, and dH in db)
// enters its product as two bfloat16 terms: 2^-17 of a term beside the output's
// own 2^-9.  H in dc and dH in dx, which da takes along, enter as three (24
// bits), and every sum is in float32 or more.
//
// H and dH come from the forward's sweep over the chunks, and from the same
// kernel run over dy and c from the sequence's end (nothing is kept from the
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
  // [batch][heads][chunks][head_dim][state_dim]: H, the state each chunk starts
  // from, and dH, the gradient of the state it ends with
  const float *states, *ends;
  float *part;  // [3][heads][batch * chunks * 4]: da, dd, ddt_bias, one per wave
};

constexpr int kHeadAhead = 4;  // heads whose steps are found together, one by each wave

template <typename T, int NT>
struct GradLds {
  static constexpr int kTerms = Terms<T, 3>::kN;
  T x[kChunk * kLd<T, (int)kPTile>], dy[kChunk * kLd<T, (int)kPTile>];
  T b[kChunk * kLd<T, NT>], c[kChunk * kLd<T, NT>];
  T h[kTerms][kPTile * kLd<T, NT>];  // H, then dH
  Steps st[kHeadAhead];
  // Sums over tokens that da needs, by wave: what is added from a token on
  // (cancelling, not cancelling) and before it; <dH, H>
  double after[4], from[4], before[4];
  float whole[4];
};

// 64 x NT values of a state on their way from global memory to LDS.  Rows and
// columns past the state's are read from the last inside it and become zeros.
template <int NT, bool kWideRows>
struct StateTile {
  static constexpr int kPer = 64 * (NT / 4) / 256;
  f32x4 v[kPer];
  __device__ __forceinline__ void fetch(const float *g, uint32_t rows, uint32_t cols) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + 256 * i, p = min(e / (NT / 4), rows - 1),
                     n = (e % (NT / 4)) * 4;
      const NSFPS_GLOBAL_SEQ float *at = (const NSFPS_GLOBAL_SEQ float *)(g + p * cols);
      if constexpr (kWideRows) {
        v[i] = *(const NSFPS_GLOBAL_SEQ f32x4 *)(at + min(n, cols - 4));
      } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) v[i][k] = at[min(n + k, cols - 1)];
      }
    }
  }
  __device__ __forceinline__ void mask(uint32_t rows, uint32_t cols) {
    if (rows >= 64 && cols >= NT) return;  // the same for all lanes
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + 256 * i, n = (e % (NT / 4)) * 4;
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)
        v[i][k] = e / (NT / 4) < rows && n + k < cols ? v[i][k] : 0.f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void put(GradLds<T, NT> &m) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + 256 * i, p = e / (NT / 4), n = (e % (NT / 4)) * 4;
      const Terms<T, 3> t = split<T, 3>(v[i]);
#pragma unroll
      for (int k = 0; k < Terms<T, 3>::kN; ++k) put_quad(m.h[k], kLd<T, NT>, p, n, t.q[k]);
    }
  }
  // <this, the state put in LDS by the same threads>: its terms add up to it
  template <typename T>
  __device__ __forceinline__ float dot(const GradLds<T, NT> &m) const {
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = threadIdx.x + 256 * i, p = e / (NT / 4), n = (e % (NT / 4)) * 4;
      f32x4 h = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = Terms<T, 3>::kN - 1; k >= 0; --k)
        h += quad_f32(quad_row(m.h[k], kLd<T, NT>, p, n));
#pragma unroll
      for (int k = 0; k < 4; ++k) d = fmaf(v[i][k], h[k], d);
    }
    return d;
  }
};

// Keeps what is read from LDS on its side of this point: without it the
// compiler reads the next products' operands ahead of these ones' until no
// register is left.
__device__ __forceinline__ void phase() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The two 32-lane halves (or, in each half, the two 16-lane quarters) added:
// the swap leaves one side's values in both places of one result and the other
// side's in the other.
__device__ __forceinline__ float add_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_quarters(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <bool kHalves>
__device__ __forceinline__ double add_sides(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
  uint32_t l[2], h[2];
  if constexpr (kHalves) {
    const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    l[0] = a[0], l[1] = a[1], h[0] = b[0], h[1] = b[1];
  } else {
    const auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    l[0] = a[0], l[1] = a[1], h[0] = b[0], h[1] = b[1];
  }
  return __builtin_bit_cast(double, ((uint64_t)h[0] << 32) | l[0]) +
         __builtin_bit_cast(double, ((uint64_t)h[1] << 32) | l[1]);
}
// over the four quads of a column (lanes l, 16 + l, 32 + l, 48 + l)
__device__ __forceinline__ float column_sum(float v) { return add_halves(add_quarters(v)); }
__device__ __forceinline__ double column_sum(double v) {
  return add_sides<true>(add_sides<false>(v));
}

// v of lane l - K of the same 16 lanes, 0 where there is none (DPP row shift)
template <int K>
__device__ __forceinline__ double row_shift(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)u, 0x110 + K, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(u >> 32), 0x110 + K, 0xf, 0xf, true);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
template <int K>
__device__ __forceinline__ float row_shift(float v) {
  return __uint_as_float(
      __builtin_amdgcn_update_dpp(0u, __float_as_uint(v), 0x110 + K, 0xf, 0xf, true));
}
// inclusive sum over lanes 0 .. l of each 16
template <typename V>
__device__ __forceinline__ V row_scan(V v) {
  v += row_shift<1>(v);
  v += row_shift<2>(v);
  v += row_shift<4>(v);
  return v + row_shift<8>(v);
}
// over the wave, in lanes 15, 31, 47 and 63
__device__ __forceinline__ float wave_sum(float v) { return column_sum(row_scan(v)); }

// Four values of a lane's column to a row of global memory.
template <typename T, bool kWideRows>
__device__ __forceinline__ void store_quad(T *dst, f32x4 v, uint32_t at, uint32_t cols) {
  if constexpr (kWideRows) {
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
constexpr int kGradGroups = sizeof(GradLds<T, NT>) <= 80 * 1024 ? 2 : 1;  // workgroups a CU

// Bound by what surrounds its products: operands are read from LDS for every
// 16 x 16 tile, states are split into three terms, and the four waves meet at
// barriers for each head.  64 sequences of up to 4,096 tokens, 8 heads of 64 x
// 64 in one group, bfloat16: 841 us; 3 of 1,001 tokens, 6 heads of 48 x 33,
// float32: 47 us.
// Work item w: chunk bc = w / groups of all sequences' and group w % groups.
// kOne: head_dim is at most 64, so a head is one tile and its loads run ahead.
template <typename T, int NT, bool kOne, bool kWideRows>
__global__ __launch_bounds__(256, (kGradGroups<T, NT>)) void k_scan_grad(ScanDev s, GradDev gr,
                                                                         uint64_t first_item,
                                                                         uint32_t work) {
  extern __shared__ __attribute__((aligned(16))) char s_raw[];
  GradLds<T, NT> &m = *(GradLds<T, NT> *)s_raw;
  constexpr int ldx = kLd<T, (int)kPTile>, ldn = kLd<T, NT>, kT3 = Terms<T, 3>::kN,
                kT2 = Terms<T, 2>::kN, kNt = NT / 16, kNb = NT / 32, kPb = (int)kPTile / 32;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
                 g = lane >> 4, l = lane & 15u;
  const uint32_t each = s.heads / s.groups;  // heads of a group
  const int own = 16 * wave + l;             // this lane's token, as i and as j
  if (blockIdx.x >= work) return;
  const uint64_t w = first_item + blockIdx.x, bc = w / s.groups;
  const uint32_t grp = (uint32_t)(w % s.groups), h0 = grp * each, h1 = h0 + each;
  const uint32_t c = (uint32_t)(bc % s.chunks), b = (uint32_t)(bc / s.chunks);
  const uint32_t len = scan_length(s, b), t0 = c * kChunk, sn = s.state_dim;
  const uint32_t out_rows = min(kChunk, s.length - t0);
  const uint32_t rows = t0 < len ? min(kChunk, len - t0) : 0u;
  // Rows past the end are zeros even where the sequence is spoiled: sums over
  // the chunk's tokens bring a NaN to all of them.
  const bool writes = (uint32_t)own < out_rows, inside = (uint32_t)own < rows;
  const uint64_t parts = (uint64_t)s.batch * s.chunks * 4;
  const auto rows_at = [&](const nsfps_rows &r) {
    return (T *)r.p + (uint64_t)b * r.batch_stride + (uint64_t)t0 * r.row_stride;
  };
  T *const db_row = rows_at(gr.db) + (uint64_t)own * gr.db.row_stride + grp * sn;
  T *const dc_row = rows_at(gr.dc) + (uint64_t)own * gr.dc.row_stride + grp * sn;
  T *const dx_row = rows_at(gr.dx) + (uint64_t)own * gr.dx.row_stride;
  T *const ddt_row = rows_at(gr.ddt) + (uint64_t)own * gr.ddt.row_stride;
  if (rows == 0) {  // past the sequence's end: zeros
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    if (writes) {
      for (uint32_t nt = 0; nt < kNt; ++nt) {
        store_quad<T, kWideRows>(db_row, z, 16 * nt + 4 * g, sn);
        store_quad<T, kWideRows>(dc_row, z, 16 * nt + 4 * g, sn);
      }
      for (uint32_t p = h0 * s.head_dim + 4 * g; p < h1 * s.head_dim; p += 16)
        store_quad<T, kWideRows>(dx_row, z, p, h1 * s.head_dim);
      for (uint32_t h = h0 + 4 * g; h < h1; h += 16) store_quad<T, false>(ddt_row, z, h, h1);
    }
    if (threadIdx.x < 12)
      for (uint32_t h = h0; h < h1; ++h)
        gr.part[((uint64_t)(threadIdx.x >> 2) * s.heads + h) * parts + bc * 4 + (threadIdx.x & 3)] =
            0.f;
    return;
  }
  const uint32_t ptiles = kOne ? 1u : s.ptiles;
  const T *const x_at = rows_at(s.x), *const dy_at = rows_at(gr.dy);
  Tile<T, (int)kPTile, kWideRows> tx, tdy;
  StateTile<NT, kWideRows> th, tdh;
  const auto fetch_xdy = [&](uint32_t h, uint32_t pt) {
    const uint32_t at = h * s.head_dim + pt * kPTile, cols = s.head_dim - pt * kPTile;
    tx.fetch(x_at + at, s.x.row_stride, rows, cols);
    tdy.fetch(dy_at + at, gr.dy.row_stride, rows, cols);
  };
  const auto state_at = [&](uint32_t h, uint32_t pt) {
    return ((((uint64_t)b * s.heads + h) * s.chunks + c) * s.head_dim + pt * kPTile) * sn;
  };
  const auto fetch_h = [&](uint32_t h, uint32_t pt) {
    th.fetch(gr.states + state_at(h, pt), s.head_dim - pt * kPTile, sn);
  };
  const auto fetch_dh = [&](uint32_t h, uint32_t pt) {
    tdh.fetch(gr.ends + state_at(h, pt), s.head_dim - pt * kPTile, sn);
  };
  // raw steps (and bias and a) of the head this wave finds the steps of; the
  // last head and token again past the end
  Raw<T, 1> raw = zero_raw<T, 1>();
  float raw_bias = 0.f, raw_a = 0.f;
  const auto fetch_raw = [&](uint32_t h) {
    const uint32_t hw = min(h + wave, h1 - 1);
    raw = raw_step<T>(s, b, hw, t0 + min(lane, rows - 1));
    raw_bias = s.dt_bias ? s.dt_bias[hw] : 0.f;
    raw_a = s.a[hw];
  };
  // the head's own parameters
  float a_h = 0.f, skip = 0.f;
  const auto fetch_params = [&](uint32_t h) {
    a_h = s.a[h];
    skip = s.d ? s.d[h] : 0.f;
  };
  {
    Tile<T, NT, kWideRows> tb, tc;
    fetch_params(h0);
    tb.fetch(rows_at(s.b) + grp * sn, s.b.row_stride, rows, sn);
    tc.fetch(rows_at(s.c) + grp * sn, s.c.row_stride, rows, sn);
    fetch_xdy(h0, 0);
    if constexpr (kOne) fetch_h(h0, 0);
    fetch_raw(h0);
    tb.put(m.b);
    tc.put(m.c);
  }
  __syncthreads();

  // S = c b^T with this wave's tokens as rows i (tiles of columns j <= its
  // own), transposed, or as columns j (tiles of rows i >= its own).  The same
  // for every head, and found again for each: it would hold 32 registers.
  const auto find_s = [&](auto as_i, f32x4(&st)[4]) __attribute__((always_inline)) {
    constexpr bool kAsI = decltype(as_i)::value;
    unrolled<kNb>([&](auto kb) __attribute__((always_inline)) {
      const Pair<T> o = pair_row(kAsI ? m.c : m.b, ldn, own, kb, g);
      unrolled<4>([&](auto t) __attribute__((always_inline)) {
        if (kAsI ? t <= (int)wave : t >= (int)wave) {
          mma_apart(st[t], pair_row(kAsI ? m.b : m.c, ldn, 16 * t + l, kb, g), o);
          settle<T>();
        }
      });
    });
  };

  f32x4 db[kNt] = {}, dc[kNt] = {};
  for (uint32_t h = h0; h < h1; ++h) {
    const Steps &sp = m.st[(h - h0) % kHeadAhead];
    phase();
    const auto put_xdy = [&] {
      tx.put(m.x);
      tdy.put(m.dy);
    };
    // W = dy x^T with this wave's tokens as rows i (kAsI) or columns j, of the
    // tile in LDS
    const auto add_w = [&](auto as_i, f32x4(&wt)[4]) __attribute__((always_inline)) {
      constexpr bool kAsI = decltype(as_i)::value;
      unrolled<kPb>([&](auto kb) __attribute__((always_inline)) {
        const Pair<T> o = pair_row(kAsI ? m.dy : m.x, ldx, own, kb, g);
        unrolled<4>([&](auto t) __attribute__((always_inline)) {
          if (kAsI ? t <= (int)wave : t >= (int)wave) {
            mma_apart(wt[t], pair_row(kAsI ? m.x : m.dy, ldx, 16 * t + l, kb, g), o);
            settle<T>();
          }
        });
      });
    };
    f32x4 w_i[4] = {}, w_j[4] = {};
    for (uint32_t pt = 0; pt < ptiles; ++pt) {
      if (!kOne && (pt || h > h0)) fetch_xdy(h, pt);
      __syncthreads();  // all are done with the head (or tile) before
      put_xdy();
      if constexpr (kOne) {
        th.mask(s.head_dim, sn);
        th.put(m);
      }
      if (pt == 0 && (h - h0) % kHeadAhead == 0) {
        chunk_steps(m.st[wave], number(raw) + raw_bias, lane < rows, raw_a);
        fetch_raw(h + kHeadAhead);
      }
      __syncthreads();
      if constexpr (kOne) fetch_dh(h, 0);
      add_w(std::true_type(), w_i);
      if constexpr (!kOne) add_w(std::false_type(), w_j);
    }

    phase();
    // ---- as rows i: G, and T's sums over j < i.  L_ij S_ij W_ij is summed in
    // float64 and rounded alike in both orientations: below, sums over rows are
    // taken from sums over columns, and what is in both must go.
    double rt = 0.0;
    {
      Terms<T, 2> g_i[4];
      f32x4 s_i[4] = {};
      find_s(std::true_type(), s_i);
      const float hi = sp.hi[own], lo = sp.lo[own];
      unrolled<4>([&](auto t) __attribute__((always_inline)) {
        f32x4 gi = {0.f, 0.f, 0.f, 0.f};
        if (t <= (int)wave) {
          const int j0 = 16 * t + 4 * g;
          const f32x4 dj = quad_of(sp.delta, j0), hj = quad_of(sp.hi, j0), lj = quad_of(sp.lo, j0);
          unrolled<4>([&](auto r_) __attribute__((always_inline)) {
            constexpr int r = decltype(r_)::value;
            const float le = exp2_fast((hi - hj[r]) + (lo - lj[r]));
            const float lw = j0 + r <= own ? le : 0.f;
            gi[r] = lw * dj[r] * w_i[t][r];
            const float tv = (lw * s_i[t][r]) * w_i[t][r];
            rt = fma((double)(j0 + r != own ? tv : 0.f), (double)dj[r], rt);
          });
        }
        g_i[t] = split<T, 2>(gi);
      });
      rt = column_sum(rt);
      unrolled<2>([&](auto kb) __attribute__((always_inline)) {
        if (2 * kb <= (int)wave) {
          unrolled<kNt>([&](auto nt) __attribute__((always_inline)) {
            const Pair<T> a = pair_col(m.b, ldn, kb, 16 * nt, g, l);
            unrolled<kT2>([&](auto k) __attribute__((always_inline)) {
              mma(dc[nt], a, Pair<T>{g_i[2 * kb].q[k], g_i[2 * kb + 1].q[k]});
            });
          });
          settle<T>();
        }
      });
    }
    phase();
    // ---- as columns j: M and G, and T's sums over i > j without delta_j
    Terms<T, 2> m_j[4];
    double u_off = 0.0;
    float diag = 0.f, dd = 0.f;
    const float delta = sp.delta[own];
    if constexpr (kOne) add_w(std::false_type(), w_j);
    {
      Terms<T, 2> g_j[4];
      f32x4 s_j[4] = {};
      find_s(std::false_type(), s_j);
      const float hj = sp.hi[own], lj = sp.lo[own];
      unrolled<4>([&](auto t) __attribute__((always_inline)) {
        f32x4 mj = {0.f, 0.f, 0.f, 0.f}, gj = mj;
        if (t >= (int)wave) {
          const int i0 = 16 * t + 4 * g;
          const f32x4 hi = quad_of(sp.hi, i0), lo = quad_of(sp.lo, i0);
          unrolled<4>([&](auto r_) __attribute__((always_inline)) {
            constexpr int r = decltype(r_)::value;
            const float le = exp2_fast((hi[r] - hj) + (lo[r] - lj));
            const float lw = i0 + r >= own ? le : 0.f, ls = lw * s_j[t][r];
            const float tv = ls * w_j[t][r];
            mj[r] = ls * delta;
            gj[r] = lw * delta * w_j[t][r];
            const bool on = i0 + r == own;  // the diagonal
            dd = on ? w_j[t][r] : dd;
            diag = on ? tv : diag;
            u_off += (double)(on ? 0.f : tv);
          });
        }
        m_j[t] = split<T, 2>(mj);
        g_j[t] = split<T, 2>(gj);
      });
      u_off = column_sum(u_off);
      diag = column_sum(diag);
      unrolled<2>([&](auto kb) __attribute__((always_inline)) {
        if (2 * kb + 1 >= (int)wave) {
          unrolled<kNt>([&](auto nt) __attribute__((always_inline)) {
            const Pair<T> a = pair_col(m.c, ldn, kb, 16 * nt, g, l);
            unrolled<kT2>([&](auto k) __attribute__((always_inline)) {
              mma(db[nt], a, Pair<T>{g_j[2 * kb].q[k], g_j[2 * kb + 1].q[k]});
            });
          });
          settle<T>();
        }
      });
    }

    phase();
    // ---- what passes through the states, 64 rows of them at a time
    const float e_i = sp.e[own], to_end = sp.end[own], w_end = delta * to_end;
    float thru = 0.f, dot = 0.f, from = 0.f;
    for (uint32_t pt = 0; pt < ptiles; ++pt) {
      const uint32_t p0 = pt * kPTile, pn = s.head_dim - p0;
      if constexpr (!kOne) {
        fetch_xdy(h, pt);
        fetch_h(h, pt);
        __syncthreads();
        put_xdy();
        th.mask(pn, sn);
        th.put(m);
        __syncthreads();
        fetch_dh(h, pt);
      }
      // H^T dy_i
      unrolled<kNt>([&](auto nt) __attribute__((always_inline)) {
        phase();
        f32x4 v = {0.f, 0.f, 0.f, 0.f}, low = v;
        unrolled<kPb>([&](auto kb) __attribute__((always_inline)) {
          const Pair<T> go = pair_row(m.dy, ldx, own, kb, g);
#pragma unroll
          for (int k = kT3 - 1; k > 0; --k) mma(low, pair_col(m.h[k], ldn, kb, 16 * nt, g, l), go);
          mma_apart(v, pair_col(m.h[0], ldn, kb, 16 * nt, g, l), go);
        });
        v += low;
        const f32x4 cv = quad_f32(quad_row(m.c, ldn, own, 16 * nt + 4 * g));
        unrolled<4>([&](auto r_) __attribute__((always_inline)) {
          constexpr int r = decltype(r_)::value;
          from = fmaf(cv[r], v[r], from);
        });
        dc[nt] += v * e_i;
      });
      __syncthreads();
      tdh.mask(pn, sn);
      dot += tdh.dot(m);
      tdh.put(m);
      __syncthreads();
      const float skip_h = skip;
      if constexpr (kOne) fetch_xdy(min(h + 1, h1 - 1), 0);  // the last again at the end
      // dH^T x_j
      unrolled<kNt>([&](auto nt) __attribute__((always_inline)) {
        phase();
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        unrolled<kPb>([&](auto kb) __attribute__((always_inline)) {
          const Pair<T> xo = pair_row(m.x, ldx, own, kb, g);
#pragma unroll
          for (int k = kT2 - 1; k >= 0; --k) mma(v, pair_col(m.h[k], ldn, kb, 16 * nt, g, l), xo);
        });
        db[nt] += v * w_end;
      });
      // dx: through the chunk, and dH b_j
      unrolled<(int)kPTile / 16>([&](auto q) __attribute__((always_inline)) {
        phase();
        f32x4 in = {0.f, 0.f, 0.f, 0.f}, thr = in, low = in;
        unrolled<2>([&](auto kb) __attribute__((always_inline)) {
          if (2 * kb + 1 >= (int)wave) {
            const Pair<T> a = pair_col(m.dy, ldx, kb, 16 * q, g, l);
            unrolled<kT2>([&](auto k) __attribute__((always_inline)) {
              mma(in, a, Pair<T>{m_j[2 * kb].q[k], m_j[2 * kb + 1].q[k]});
            });
            settle<T>();
          }
        });
        unrolled<kNb>([&](auto kb) __attribute__((always_inline)) {
          const Pair<T> bo = pair_row(m.b, ldn, own, kb, g);
#pragma unroll
          for (int k = kT3 - 1; k > 0; --k) mma(low, pair_row(m.h[k], ldn, 16 * q + l, kb, g), bo);
          mma_apart(thr, pair_row(m.h[0], ldn, 16 * q + l, kb, g), bo);
        });
        thr += low;
        const f32x4 xv = quad_f32(quad_row(m.x, ldx, own, 16 * q + 4 * g));
        const f32x4 gv = quad_f32(quad_row(m.dy, ldx, own, 16 * q + 4 * g));
        f32x4 o;
        unrolled<4>([&](auto r_) __attribute__((always_inline)) {
          constexpr int r = decltype(r_)::value;
          thru = fmaf(xv[r], thr[r], thru);
          const float v = fmaf(skip_h, gv[r], fmaf(w_end, thr[r], in[r]));
          o[r] = inside ? v : 0.f;
        });
        if (writes) store_quad<T, kWideRows>(dx_row + h * s.head_dim + p0, o, 16 * q + 4 * g, pn);
      });
    }
    phase();
    if constexpr (kOne) fetch_h(min(h + 1, h1 - 1), 0);
    thru = column_sum(thru) * to_end;  // per delta_j
    from = column_sum(from) * e_i;
    dot = wave_sum(dot);

    // ---- the exponents: sums over the chunk's tokens from each on, and before
    // it.  The 16 tokens of a wave are lanes l of each quarter.
    const double after = rt - (double)delta * u_off;  // cancels over the tokens
    const double mine = (double)delta * thru;
    const double sum_after = row_scan(after), sum_from = row_scan((double)from),
                 sum_before = row_scan(mine);
    if (lane == 15) {
      m.after[wave] = sum_after;
      m.from[wave] = sum_from;
      m.before[wave] = sum_before;
      m.whole[wave] = dot;
    }
    __syncthreads();
    double a_on = after - sum_after, f_on = (double)from - sum_from, before = sum_before - mine;
    unrolled<4>([&](auto o) __attribute__((always_inline)) {
      if (o >= (int)wave) a_on += m.after[o], f_on += m.from[o];
      if (o < (int)wave) before += m.before[o];
    });
    const float whole =
        exp2_fast(sp.total) * (m.whole[0] + m.whole[1] + m.whole[2] + m.whole[3]);
    const float da = (float)(a_on + f_on + before) + whole;
    const float ddt = fmaf(a_h, da, (float)u_off + diag + thru) * sp.sig[own];
    const float o[1] = {inside ? ddt : 0.f};
    if (writes && g == 0) store_f32<T, 1>(ddt_row + h, o);
    // one quarter each: da, ddt_bias; dd is on the diagonal's lanes
    const float sums = (float)row_scan(g == 0 ? (double)delta * da : (double)ddt);
    dd = wave_sum(dd);
    float *part = gr.part + (uint64_t)h * parts + bc * 4 + wave;
    if (l == 15) {
      if (g == 0) part[0] = sums;
      if (g == 1) part[2 * s.heads * parts] = sums;
      if (g == 2) part[s.heads * parts] = dd;
    }
    fetch_params(min(h + 1, h1 - 1));
  }
  if (writes) {
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    unrolled<kNt>([&](auto nt) __attribute__((always_inline)) {
      store_quad<T, kWideRows>(db_row, inside ? db[nt] : z, 16 * nt + 4 * g, sn);
      store_quad<T, kWideRows>(dc_row, inside ? dc[nt] : z, 16 * nt + 4 * g, sn);
    });
  }
}

// One workgroup per head and parameter: the chunks' parts in a fixed order.
// 8 heads of 4,096 chunks: 4.6 us, about a launch.
__global__ __launch_bounds__(1024) void k_scan_grad_join(const float *__restrict__ part,
                                                         uint64_t count, uint32_t heads, float *da,
                                                         float *dd, float *ddt_bias) {
  constexpr uint32_t kAhead = 8;
  __shared__ double s_sum[16];
  float *const out[3] = {da, dd, ddt_bias};
  const uint32_t h = blockIdx.x, k = blockIdx.y;
  const float *p = part + ((uint64_t)k * heads + h) * count;
  double sum = 0.0;
  for (uint64_t i = threadIdx.x; i < count; i += 1024 * kAhead) {
    float v[kAhead];
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) v[j] = p[min(i + 1024 * j, count - 1)];
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) sum += i + 1024 * j < count ? (double)v[j] : 0.0;
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0 && out[k]) {
    double all = 0.0;
    for (int w = 0; w < 16; ++w) all += s_sum[w];
    out[k][h] = (float)all;
  }
}

uint64_t part_bytes(const nsfps_scan_args &a) {
  return round256(48 * a.batch * a.heads * host_ceil_div(a.length, kChunk));
}

}  // namespace

namespace {
uint64_t chunk_states_bytes(const ScanDev &s) {
  return round256(4ull * s.batch * s.heads * s.chunks * s.head_dim * s.state_dim);
}
}  // namespace

uint64_t scan_grad_bytes(const nsfps_scan_args &a) {
  const ScanDev s = scan_dev(a);
  return 2 * chunk_states_bytes(s) + part_bytes(a) + carry_bytes(s);
}

hipError_t launch_scan_grad(const nsfps_scan_args &a, const nsfps_scan_grads &g, hipStream_t st) {
  const ScanDev s = scan_dev(a);
  char *const ws = (char *)a.workspace;
  float *const states = (float *)ws, *const ends = (float *)(ws + chunk_states_bytes(s));
  char *const carry = ws + 2 * chunk_states_bytes(s) + part_bytes(a);
  GradDev d = {};
  d.dy = g.dy;
  d.dx = g.dx;
  d.db = g.db;
  d.dc = g.dc;
  d.ddt = g.ddt;
  d.states = states;
  d.ends = ends;
  d.part = (float *)(ws + 2 * chunk_states_bytes(s));
  const uint64_t parts = a.batch * s.chunks, work = parts * s.groups;
  if (work) {
    hipError_t e = launch_states(a, s, s.x, s.b, states, false, carry, st);
    if (e == hipSuccess) e = launch_states(a, s, d.dy, s.c, ends, true, carry, st);
    if (e != hipSuccess) return e;
    const bool wide = scan_wide(a, {&a.x, &a.b, &a.c, &g.dy, &g.dx, &g.db, &g.dc});
    e = scan_by_type(a.dtype, a.state_dim, wide, [&](auto t, auto n, auto w) {
      using T = decltype(t);
      constexpr int NT = decltype(n)::value;
      constexpr bool kWideRows = decltype(w)::value;
      constexpr size_t lds = sizeof(GradLds<T, NT>);
      static_assert(lds <= 160 * 1024, "LDS");
      const auto go = [&](auto kernel) {
        const hipError_t e2 = hipFuncSetAttribute(
            (const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e2 != hipSuccess) return e2;
        constexpr uint64_t kLaunch = 1u << 23;  // workgroups of a launch: fewer than 2^32 threads
        for (uint64_t at = 0; at < work; at += kLaunch) {
          const uint32_t some = (uint32_t)std::min(kLaunch, work - at);
          kernel<<<some, 256, lds, st>>>(s, d, at, some);
        }
        return hipGetLastError();
      };
      return s.ptiles == 1 ? go(k_scan_grad<T, NT, true, kWideRows>)
                           : go(k_scan_grad<T, NT, false, kWideRows>);
    });
    if (e != hipSuccess) return e;
  }
  k_scan_grad_join<<<dim3(a.heads, 3), 1024, 0, st>>>(d.part, 4 * parts, a.heads, g.d_da, g.d_dd,
                                                     g.d_ddt_bias);
  return hipGetLastError();
}

hipError_t preload_scan_grad_kernels() {
  return func_attributes(k_scan_grad<bf16, 64, true, true>, k_scan_grad_join);
}

}  // namespace nsfps
