// Device helpers of the sequence operators: the two storage types, vectors of
// them, and the exponential.  Contraction to FMA is wanted here (a sum of
// products has no order of operations to reproduce, and an FMA rounds once),
// so the operators' files switch it on.
#pragma once

#include "nsfps_sequence.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#if defined(__HIP_DEVICE_COMPILE__)
#define NSFPS_GLOBAL_SEQ __attribute__((address_space(1)))
#else
#define NSFPS_GLOBAL_SEQ
#endif

namespace nsfps {
namespace seq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct bf16 {
  uint16_t u;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __uint_as_float((uint32_t)v.u << 16); }

// Nearest even, as the hardware converts (NaN stays NaN).
__device__ __forceinline__ uint16_t bf16_bits(float v) {
  const __bf16 h = (__bf16)v;
  return __builtin_bit_cast(uint16_t, h);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) {
  return bf16{bf16_bits(v)};
}

// V elements at p, p aligned to V elements, as loaded (a load whose values are
// converted where it stands is waited for there) ...
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * (int)sizeof(T), kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];
};
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T *p) {
  const NSFPS_GLOBAL_SEQ T *g = (const NSFPS_GLOBAL_SEQ T *)p;
  Raw<T, V> o;
  if constexpr (Raw<T, V>::kBytes == 16) {
    const u32x4 t = *(const NSFPS_GLOBAL_SEQ u32x4 *)g;
    o.w[0] = t.x, o.w[1] = t.y, o.w[2] = t.z, o.w[3] = t.w;
  } else if constexpr (Raw<T, V>::kBytes == 8) {
    const u32x2 t = *(const NSFPS_GLOBAL_SEQ u32x2 *)g;
    o.w[0] = t.x, o.w[1] = t.y;
  } else if constexpr (Raw<T, V>::kBytes == 4) {
    o.w[0] = *(const NSFPS_GLOBAL_SEQ uint32_t *)g;
  } else {
    static_assert(Raw<T, V>::kBytes == 2, "vector width");
    o.w[0] = *(const NSFPS_GLOBAL_SEQ uint16_t *)g;
  }
  return o;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> zero_raw() {
  Raw<T, V> o;
#pragma unroll
  for (int i = 0; i < Raw<T, V>::kWords; ++i) o.w[i] = 0u;
  return o;
}
// ... and as numbers
template <typename T, int V>
__device__ __forceinline__ void numbers(const Raw<T, V> &r, float (&o)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (sizeof(T) == 4)
      o[i] = __uint_as_float(r.w[i]);
    else
      o[i] = __uint_as_float((i & 1) ? (r.w[i / 2] & 0xffff0000u) : (r.w[i / 2] << 16));
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_f32(const T *p, float (&o)[V]) {
  numbers<T, V>(load_raw<T, V>(p), o);
}
template <typename T, int V>
__device__ __forceinline__ void store_f32(T *p, const float (&o)[V]) {
  NSFPS_GLOBAL_SEQ T *g = (NSFPS_GLOBAL_SEQ T *)p;
  constexpr int kWords = V * (int)sizeof(T) / 4;
  if constexpr (kWords >= 1) {
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(o[i]);
      else
        w[i] = (uint32_t)bf16_bits(o[2 * i]) | ((uint32_t)bf16_bits(o[2 * i + 1]) << 16);
    }
    if constexpr (kWords == 4) {
      u32x4 t;
      t.x = w[0], t.y = w[1], t.z = w[2], t.w = w[3];
      *(NSFPS_GLOBAL_SEQ u32x4 *)g = t;
    } else if constexpr (kWords == 2) {
      u32x2 t;
      t.x = w[0], t.y = w[1];
      *(NSFPS_GLOBAL_SEQ u32x2 *)g = t;
    } else {
      *(NSFPS_GLOBAL_SEQ uint32_t *)g = w[0];
    }
  } else {
    if constexpr (sizeof(T) == 4)
      *(NSFPS_GLOBAL_SEQ uint32_t *)g = __float_as_uint(o[0]);
    else
      *(NSFPS_GLOBAL_SEQ uint16_t *)g = bf16_bits(o[0]);
  }
}

// Elements of a 16-byte load.
template <typename T>
constexpr int kWide = 16 / (int)sizeof(T);

constexpr float kLog2e = 1.44269504088896340736f;

// 2^x (v_exp_f32: within an ulp; results below the normal range become 0)
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }
constexpr float kLn2 = 0.693147180559945309417f, kLn2Low = -1.90465429995776e-9f;
// exp(x) is 2^p of the float32 product p = x log2(e) times 1 + (x - p ln 2): what
// the product's rounding took, which would else put |x| 2^-24 into the result.
// (float32 ln 2 is off by 2^-28 of itself, kLn2Low is the rest.)
__device__ __forceinline__ float exp_rest(float x, float p) {
  return fmaf(-p, kLn2Low, fmaf(-p, kLn2, x));
}
// exp(x + low), low a few bits below x, to 2^-22 of itself.  Arguments of -200
// and less give 0, NaN stays; for x up to 88.
__device__ __forceinline__ float exp_f32(float x, float low = 0.f) {
  const float t = x < -200.f ? -200.f : x, p = t * kLog2e, y = exp2_fast(p);
  return fmaf(y, exp_rest(t, p) + low, y);
}
// sig = 1 / (1 + exp(-x)), rest = 1 / (1 + exp(x)), each to a few units of its
// own last place while sig is not 0; below x = -88 both are 0.  The bounds keep
// an infinity from meeting a 0.
struct Logistic {
  float sig, rest;
};
__device__ __forceinline__ Logistic logistic(float x) {
  const float t = __builtin_amdgcn_fmed3f(-x, -200.f, 200.f), p = t * kLog2e;
  const float e = exp2_fast(p) * (1.f + exp_rest(t, p)), sig = rcp_fast(1.f + e);
  return Logistic{sig, fminf(e, 3e38f) * sig};
}
__device__ __forceinline__ float sigmoid(float x) { return logistic(x).sig; }
// The same without the remainder, to |x| 2^-23 of itself (2^-16 at most): for
// results that are rounded to 8 bits next.
__device__ __forceinline__ float sigmoid_8bit(float x) {
  return rcp_fast(1.f + exp2_fast(-x * kLog2e));
}
// log(1 + exp(x)) without overflow, and its derivative; -infinity gives 0, 0
__device__ __forceinline__ float softplus(float x, float &slope) {
  const float e = exp_f32(-fabsf(x)), r = rcp_fast(1.f + e);
  slope = x < 0.f ? e * r : r;
  return fmaxf(x, 0.f) + log1pf(e);
}

// f(0), f(1) .. f(N - 1) with the index a constant: arrays of registers are
// indexed by constants whatever the optimizer's order of passes.  (A loop that
// is unrolled late leaves its arrays to be merged into one wide value, which
// is then copied whole for every element that changes.)
template <typename F, int... I>
__device__ __forceinline__ void unrolled_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled_of(f, std::make_integer_sequence<int, N>());
}

// Waits for this wave's loads.  Before a loop that fetches ahead: values loaded
// before it would else be waited for at their first use inside, every time
// round, and the loads ahead with them.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

__device__ __forceinline__ uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

}  // namespace seq

inline uint64_t host_ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Rows whose start and strides keep 16-byte loads of `size`-byte elements aligned.
inline bool rows_wide(const nsfps_rows &r, uint32_t size) {
  const uint64_t v = 16 / size;
  return (uintptr_t)r.p % 16 == 0 && r.batch_stride % v == 0 && r.row_stride % v == 0;
}

}  // namespace nsfps
