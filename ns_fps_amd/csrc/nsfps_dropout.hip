// Dropout onto a residual: y = residual + (kept ? x / (1 - p) : 0), the mask
// made where it is used.
//
// Eight channels of a row share one call of the generator, Philox 4x32-10
// (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// 2011): ten rounds of two 32 x 32 bit products, whose high words are mixed
// into the other pair of words.  16 bits a value are enough for a drop
// probability in 65536ths and halve the generator's work, which at a quarter of
// the vector rate for products would else weigh more than the memory.
//
// Memory is the bound: 64 x 4,096 rows of 640 bfloat16, three quarters of them
// inside, onto a residual 150 us, its gradient 132, one after the other 286: 5.0 TB/s
// read and written.
#include "nsfps_launch.h"
#include "nsfps_seq_device.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

struct DropDev {
  uint32_t length, channels, blocks;  // blocks of eight channels a row
  uint32_t drop;                      // in 65536ths
  float factor;
  uint64_t work;  // blocks of all rows
  nsfps_rows x, residual, y;
  const uint64_t *seed;
  const int32_t *lengths;
};

struct Key {
  uint32_t k0, k1, c2, c3;
};

// The bits of which of a block's eight values are kept.
__device__ __forceinline__ uint32_t kept(const Key &key, uint32_t block, uint32_t row,
                                         uint32_t drop) {
  uint32_t c0 = block, c1 = row, c2 = key.c2, c3 = key.c3, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
    m |= (bits >= drop ? 1u : 0u) << i;
  }
  return m;
}

// One rounding; what is dropped may hold anything.
__device__ __forceinline__ float dropped(float x, float r, bool keep, float factor) {
  return fmaf(keep ? x : 0.f, factor, r);
}

// A lane writes the places that it has read: y may be the rows of x or residual.
// kWideRows: a lane has a block of eight values, in 16-byte accesses (the case above
// 286 us, 684 the other way).  Else a wave makes the masks of 64 blocks, a lane each,
// and takes their 512 values 64 neighbours at a time, each lane asking for the mask of
// its value's block (16,384 rows of 323 float32: 10.8 us, 3.9 TB/s).
template <typename T, bool kWideRows>
__global__ __launch_bounds__(256) void k_dropout(DropDev a) {
  const uint64_t seed = a.seed[0], call = a.seed[1];
  const Key key{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)call, (uint32_t)(call >> 32)};
  if constexpr (kWideRows) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < a.work;
         i += (uint64_t)gridDim.x * 256) {
      const uint32_t row = (uint32_t)(i / a.blocks), block = (uint32_t)(i % a.blocks);
      const uint32_t b = row / a.length, t = row % a.length;
      bool inside = true;
      if (a.lengths) {
        const int32_t n = a.lengths[b];
        inside = n > 0 && t < (uint32_t)n;
      }
      constexpr int V = kWide<T>;
      const T *const x = (const T *)a.x.p + b * a.x.batch_stride + t * a.x.row_stride + 8ull * block;
      const T *const r = (const T *)a.residual.p + b * a.residual.batch_stride +
                         t * a.residual.row_stride + 8ull * block;
      T *const y = (T *)a.y.p + b * a.y.batch_stride + t * a.y.row_stride + 8ull * block;
      Raw<T, V> xr[8 / V], rr[8 / V];
#pragma unroll
      for (int j = 0; j < 8 / V; ++j) {
        xr[j] = rr[j] = zero_raw<T, V>();
        if (inside) xr[j] = load_raw<T, V>(x + j * V);
        if (inside && a.residual.p) rr[j] = load_raw<T, V>(r + j * V);
      }
      const uint32_t mask = kept(key, block, row, a.drop);
#pragma unroll
      for (int j = 0; j < 8 / V; ++j) {
        float xv[V], rv[V], o[V];
        numbers<T, V>(xr[j], xv);
        numbers<T, V>(rr[j], rv);
#pragma unroll
        for (int k = 0; k < V; ++k)
          o[k] = dropped(xv[k], rv[k], mask >> (j * V + k) & 1, a.factor);
        store_f32<T, V>(y + j * V, o);
      }
    }
  } else {
    const uint32_t lane = threadIdx.x & 63u, spans = ceil_div(a.blocks, 64);
    const uint64_t waves = a.work * spans;  // work: rows
    for (uint64_t i = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < waves;
         i += (uint64_t)gridDim.x * 4) {
      const uint32_t row = (uint32_t)(i / spans), block0 = (uint32_t)(i % spans) * 64;
      const uint32_t b = row / a.length, t = row % a.length;
      bool inside = true;
      if (a.lengths) {
        const int32_t n = a.lengths[b];
        inside = n > 0 && t < (uint32_t)n;
      }
      const T *const x = (const T *)a.x.p + b * a.x.batch_stride + t * a.x.row_stride;
      const T *const r = (const T *)a.residual.p + b * a.residual.batch_stride +
                         t * a.residual.row_stride;
      T *const y = (T *)a.y.p + b * a.y.batch_stride + t * a.y.row_stride;
      float xv[8][1], rv[8][1];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t c = 8 * block0 + 64 * j + lane;
        xv[j][0] = rv[j][0] = 0.f;
        if (inside && c < a.channels) {
          load_f32<T, 1>(x + c, xv[j]);
          if (a.residual.p) load_f32<T, 1>(r + c, rv[j]);
        }
      }
      const uint32_t mask = kept(key, block0 + lane, row, a.drop);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t c = 8 * block0 + 64 * j + lane;
        const bool keep = (uint32_t)__shfl((int)mask, 8 * j + lane / 8, 64) >> (lane % 8) & 1;
        const float o[1] = {dropped(xv[j][0], rv[j][0], keep, a.factor)};
        if (c < a.channels) store_f32<T, 1>(y + c, o);
      }
    }
  }
}

}  // namespace

hipError_t launch_dropout(const nsfps_dropout_args &a, hipStream_t st) {
  DropDev d = {};
  d.length = (uint32_t)a.length;
  d.channels = a.channels;
  d.blocks = (a.channels + 7) / 8;
  d.drop = (uint32_t)std::lrint((double)a.p * 65536.);
  d.factor = d.drop < 65536 ? (float)(65536. / (65536. - d.drop)) : 0.f;
  d.x = a.x;
  d.residual = a.residual;
  d.y = a.y;
  d.seed = a.d_seed;
  d.lengths = a.d_lengths;
  const uint64_t rows = a.batch * a.length;
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2;
  const bool wide = a.channels % 8 == 0 && rows_wide(a.x, size) && rows_wide(a.y, size) &&
                    (!a.residual.p || rows_wide(a.residual, size));
  d.work = wide ? rows * d.blocks : rows;
  const uint64_t groups = wide ? host_ceil_div(d.work, 256)
                               : host_ceil_div(rows * host_ceil_div(d.blocks, 64), 4);
  const uint32_t grid = (uint32_t)std::min<uint64_t>(1u << 20, groups);
  const auto go = [&](auto t) {
    using T = decltype(t);
    if (wide)
      k_dropout<T, true><<<grid, 256, 0, st>>>(d);
    else
      k_dropout<T, false><<<grid, 256, 0, st>>>(d);
    return hipGetLastError();
  };
  return a.dtype == NSFPS_F32 ? go(float()) : go(bf16());
}

hipError_t preload_dropout_kernels() { return func_attributes(k_dropout<bf16, true>); }

}  // namespace nsfps
