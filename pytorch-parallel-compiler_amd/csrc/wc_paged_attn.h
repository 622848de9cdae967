// What the kernels of attention over a paged cache share: numbers as planes of 16-bit values, pieces of rows in registers.
#pragma once

#include "wc_paged.h"

namespace wc {

constexpr float kLog2e = 1.4426950408889634f;

// exp2 of a difference of scores; a part that holds nothing has m = -infinity
__device__ __forceinline__ float weight2(float m, float top) { return __builtin_amdgcn_exp2f(m - top); }
__device__ __forceinline__ float finite_top(float m) { return m == -INFINITY ? 0.f : m; }

template <typename MT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<MT, f16>::value) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {static_cast<f16>(a), static_cast<f16>(b)};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    return pack_bf16x2(a, b);
  }
}
template <typename MT>
__device__ __forceinline__ float unpack_lo(uint32_t v) {
  if constexpr (std::is_same<MT, f16>::value)
    return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(v)));
  else
    return bf16_lo(v);
}
template <typename MT>
__device__ __forceinline__ float unpack_hi(uint32_t v) {
  if constexpr (std::is_same<MT, f16>::value)
    return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(v >> 16)));
  else
    return bf16_hi(v);
}
// 8 floats as N planes of 16-bit values whose sum they are
template <typename MT, int N>
__device__ __forceinline__ void planes(const float (&v)[8], u32x4 (&out)[N]) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = v[e];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = pack2<MT>(f[2 * e], f[2 * e + 1]);
      out[n][e] = w;
      if (n + 1 < N) {
        f[2 * e] -= unpack_lo<MT>(w);
        f[2 * e + 1] -= unpack_hi<MT>(w);
      }
    }
}

// 8 weights >= 0 as N planes that leave out at most 2^-23 of them (two fp16 ones: 2^-21), all over 0 where the weight
// is: each but the last is what 16 bits hold of a value just under what is left, so that an infinite value in V takes the
// sum to its infinity and not, by 0 or the other sign, to NaN.
template <typename MT, int N>
__device__ __forceinline__ void weight_planes(const float (&p)[8], u32x4 (&out)[N]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a = p[2 * e], b = p[2 * e + 1];
    constexpr float under = 0x1.fffffep-1f;
#pragma unroll
    for (int n = 0; n + 1 < N; ++n) {
      uint32_t w;
      if constexpr (std::is_same<MT, f16>::value)
        w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a * under, b * under));
      else
        w = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b * under), __builtin_bit_cast(uint32_t, a * under), 0x07060302u);
      out[n][e] = w;
      a -= unpack_lo<MT>(w);
      b -= unpack_hi<MT>(w);
    }
    out[N - 1][e] = pack2<MT>(a, b);
  }
}

template <int B>
struct Raw {
  typedef uint32_t type __attribute__((ext_vector_type(B / 4)));
};
template <>
struct Raw<4> {
  typedef uint32_t type;
};
template <typename R>
__device__ __forceinline__ uint32_t dword(const R& r, int i) {
  if constexpr (sizeof(R) == 4)
    return r;
  else
    return r[i];
}
template <typename R>
__device__ __forceinline__ void clear(R& r) {
  r = R(0u);
}

// the sum of v over the lanes before this one
__device__ __forceinline__ int before(int v, int lane) {
  int sum = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(sum, off, 64);
    if (lane >= off) sum += up;
  }
  return sum - v;
}
}  // namespace wc
