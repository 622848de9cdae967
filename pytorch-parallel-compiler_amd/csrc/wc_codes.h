// 8-bit codes of rows of values: scale = max(max |x| / 127, 2^-126) (one unit less for fp32's largest value), code =
// x / scale to the nearest, ties to even.  The quotient is never formed: c = x * (1 / scale) to the nearest is off by at
// most one, and then only next to a half; the remainder x - c scale is exact (one fused multiply-add whose result fits 24
// bits) and its place against scale / 2 puts c right, for the lanes that have such a value.  The code is so a
// function of x and scale alone.
#pragma once

#include "wc_common.h"

namespace wc {

// the scale of a row whose largest magnitude, as the bits of a float, is `top` (finite)
__device__ __forceinline__ float row_scale(uint32_t top) {
  constexpr float kMost = 0x1.020406p121f;      // the largest scale: 127 of the next one round to infinity in fp32
  return fminf(fmaxf(__builtin_bit_cast(float, top) / 127.f, 0x1p-126f), kMost);
}

// Codes whose `off` is beyond this times the scale are made again by code8_near_half: 2^-15 covers the product's rounding
// and inv's, 2^-22 of a quotient of up to 127.
constexpr float kNearHalf = 0.5f - 0x1p-15f;

// x / scale to the nearest as the low byte of the result, by adding 1.5 2^23 (after which a float's last bit is 1), and
// how far that is from x
constexpr float kRound = 0x1.8p23f;
__device__ __forceinline__ uint32_t code8(float x, float scale, float inv, float& off) {
  const float c = fmaf(x, inv, kRound);
  off = fabsf(fmaf(kRound - c, scale, x));
  return __builtin_bit_cast(uint32_t, c);
}
// the code of a value whose quotient may be next to a half
__device__ __forceinline__ uint32_t code8_near_half(float x, float scale, float inv) {
  float c = fmaf(x, inv, kRound) - kRound;
  const float r = fmaf(-c, scale, x), half = 0.5f * scale;
  const bool odd = static_cast<int>(c) & 1;
  if (r > half || (r == half && odd))
    c += 1.f;
  else if (r < -half || (r == -half && odd))
    c -= 1.f;
  return __builtin_bit_cast(uint32_t, c + kRound);
}

}  // namespace wc
