// Products with weights of 4 bits: y = x W^T + bias, W[o, k] = scale[o, g] (code[o, k] - zero[o, g]), g = k / group.
//
// For the few rows of x that answering token by token has, the weights' bytes bound it: half a byte a weight against
// 2 flops a row.  So the weights are read once, as whole kilobytes per wave (a tile of 16 output rows x 128 columns
// is laid out in the order in which the lanes want it), and all rows of x meet them there, 16 to an MFMA tile.
//
//   y = sum_g scale_g (sum_k code x - zero_g sum_k x)
//
// The codes enter the product without their scale, as whole numbers in 16 bits, and the scale multiplies the fp32 sum
// of each group.  A nibble becomes a number by the bits above it: 0x4300 | code is 128 + code in bf16, 0x6400 | code
// is 1024 + code in fp16, two to an instruction.  fp16 then takes 1024 + zero off (exact); bf16 has no packed
// subtraction, so there the sum of x, by one more product with ones, takes (128 + zero) sum_k x off, whose
// rounding in fp32 is 2^-24 of 128 |sum x|.  fp32 goes as three bf16 planes of x (every bit of it down to 2^-110)
// against codes converted to bf16, without the 128.  A row of x with an infinity or NaN gives NaN in bf16 and fp32.
//
// The columns are dealt to the waves of a workgroup, which add their sums up through LDS at the end.
#include <algorithm>

#include "wc_common.h"
#include "wc_serve_abi.h"

namespace wc {
namespace {

struct Linear4 {
  const char *x, *scales, *bias;
  const uint8_t *codes, *zeros;
  char* y;
  int64_t xn, xo, xi;
  int32_t m, o, k, otiles, ktiles, steps_log2, m0;    // steps: 32-column products per group
  FastDiv by_rows, by_wg;                             // rows_inner; workgroups per model
};

template <typename T>
struct alignas(16) Eight {
  T v[8];
};
template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

// 8 codes as 16-bit numbers with 128 (bf16) or 1024 (fp16) added, or exact bf16 (fp32)
template <typename T>
__device__ __forceinline__ u32x4 numbers(uint32_t w) {
  u32x4 r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r[e] = pack_bf16x2(static_cast<float>((w >> (4 * e)) & 15u), static_cast<float>((w >> (4 * e + 16)) & 15u));
  } else {
    constexpr uint32_t kOver = std::is_same<T, bf16>::value ? 0x43004300u : 0x64006400u;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = ((w >> (4 * e)) & 0x000f000fu) | kOver;
  }
  return r;
}

// MT, RT: tiles of 16 rows of x and of 16 output rows; AL: rows of x are whole 16-byte vectors
template <typename T, int MT, int RT, int NW, bool AL>
__global__ __launch_bounds__(NW * 64) void linear4_kernel(Linear4 a) {
  constexpr bool kF32 = sizeof(T) == 4, kF16 = std::is_same<T, f16>::value;
  constexpr int NX = kF32 ? 3 : 1;                     // planes of x
  typedef typename std::conditional<kF16, f16, bf16>::type NT;
  extern __shared__ float lds[];                       // [NW][RT * 16][MT * 16]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const uint32_t model = fdiv(blockIdx.x, a.by_wg), ot0 = (blockIdx.x - model * a.by_wg.d) * RT;
  const int row0 = a.m0 + blockIdx.y * MT * 16;
  const int groups = a.ktiles << (2 - a.steps_log2);   // stored groups of a row

  const T* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const uint32_t r = std::min(row0 + t * 16 + j, a.m - 1);      // rows past the last only fill their own columns
    const uint32_t outer = fdiv(r, a.by_rows);
    x[t] = reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (r - outer * a.by_rows.d) * a.xi;
  }
  const u32x4* codes[RT];
  int64_t meta[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int64_t ot = static_cast<int64_t>(model) * a.otiles + std::min<int>(ot0 + t, a.otiles - 1);
    codes[t] = reinterpret_cast<const u32x4*>(a.codes) + ot * a.ktiles * 64 + lane;
    meta[t] = ot * groups * 16;
  }

  f32x4 acc[RT][MT] = {};
  f32x4 part[RT][MT] = {};
  f32x4 ones[MT] = {};
  const u32x4 one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  u32x4 next[RT];
  if (wave < a.ktiles)
#pragma unroll
    for (int t = 0; t < RT; ++t) next[t] = codes[t][wave * 64];
  for (int kt = wave; kt < a.ktiles; kt += NW) {
    u32x4 w[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) w[t] = next[t];
    if (kt + NW < a.ktiles)
#pragma unroll
      for (int t = 0; t < RT; ++t) next[t] = codes[t][(kt + NW) * 64];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k0 = kt * 128 + q * 32 + g * 8;
      const int grp = (kt * 4 + q) >> a.steps_log2;
      const bool last = ((q + 1) & ((1 << a.steps_log2) - 1)) == 0;
      u32x4 xf[MT][NX];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (!kF32) {
          u32x4 v = {};
          if constexpr (AL) {
            if (k0 < a.k) v = *reinterpret_cast<const u32x4*>(x[t] + k0);
          } else {
            Eight<T> s;
#pragma unroll
            for (int e = 0; e < 8; ++e) s.v[e] = k0 + e < a.k ? x[t][k0 + e] : static_cast<T>(0.f);
            v = __builtin_bit_cast(u32x4, s);
          }
          xf[t][0] = v;
        } else {
          float s[8];
          if constexpr (AL) {
            f32x4 lo = {}, hi = {};
            if (k0 < a.k) lo = *reinterpret_cast<const f32x4*>(x[t] + k0);
            if (k0 + 4 < a.k) hi = *reinterpret_cast<const f32x4*>(x[t] + k0 + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = lo[e], s[4 + e] = hi[e];
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = k0 + e < a.k ? x[t][k0 + e] : 0.f;
          }
          uint4 pl[3];
          split_planes(s, pl);
#pragma unroll
          for (int n = 0; n < 3; ++n) xf[t][n] = __builtin_bit_cast(u32x4, pl[n]);
        }
      }
      if constexpr (!kF16)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = NX - 1; n >= 0; --n)
            ones[t] = mma16<bf16>(__builtin_bit_cast(bf16x8, one), __builtin_bit_cast(bf16x8, xf[t][n]), ones[t]);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        u32x4 c = numbers<T>(w[r][q]);
        if constexpr (kF16) {
          typedef _Float16 h2 __attribute__((ext_vector_type(2)));
          const f16 z = static_cast<f16>(1024.f + (a.zeros ? a.zeros[meta[r] + grp * 16 + j] : 8));
          const h2 zz = {z, z};
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, static_cast<uint32_t>(c[e])) - zz);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = NX - 1; n >= 0; --n)
            part[r][t] = mma16<NT>(__builtin_bit_cast(bf16x8, c), __builtin_bit_cast(bf16x8, xf[t][n]), part[r][t]);
      }
      if (last) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int64_t at = meta[r] + grp * 16 + g * 4;
          const Four<T> sc = *reinterpret_cast<const Four<T>*>(reinterpret_cast<const T*>(a.scales) + at);
          float z[4] = {8.f, 8.f, 8.f, 8.f};
          if (!kF16 && a.zeros) {
            const uint32_t zw = *reinterpret_cast<const uint32_t*>(a.zeros + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = static_cast<float>((zw >> (8 * e)) & 255u);
          }
#pragma unroll
          for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float s = part[r][t][e];
              if constexpr (!kF16) s -= (z[e] + (kF32 ? 0.f : 128.f)) * ones[t][e];
              acc[r][t][e] += to_f32(sc.v[e]) * s;
            }
            part[r][t] = f32x4{};
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) ones[t] = f32x4{};
      }
    }
  }

  // lane: rows 4 g + e of an output tile, row j of x
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        lds[(wave * MT * 16 + t * 16 + j) * (RT * 16) + r * 16 + g * 4 + e] = acc[r][t][e];
  __syncthreads();
  T* y = reinterpret_cast<T*>(a.y) + static_cast<int64_t>(model) * a.m * a.o;
  for (int i = threadIdx.x; i < MT * 16 * RT * 16; i += NW * 64) {
    const int row = row0 + i / (RT * 16), o = ot0 * 16 + i % (RT * 16);
    if (row >= a.m || o >= a.o) continue;
    float s = 0.f;
    for (int w = 0; w < NW; ++w) s += lds[w * MT * 16 * RT * 16 + i];
    if (a.bias) s += to_f32(reinterpret_cast<const T*>(a.bias)[static_cast<int64_t>(model) * a.o + o]);
    y[static_cast<int64_t>(row) * a.o + o] = from_f32<T>(s);
  }
}

template <typename T, int MT, int RT, int NW>
void launch(Linear4 a, int64_t n, bool al, hipStream_t s) {
  const int64_t per = cdiv(a.otiles, RT);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(per));
  const size_t lds = static_cast<size_t>(NW) * RT * 16 * MT * 16 * sizeof(float);
  // grids of at most 65535 tiles of rows
  for (int64_t m0 = 0; m0 < a.m; m0 += 65535ll * MT * 16) {
    a.m0 = static_cast<int32_t>(m0);
    const dim3 grid(static_cast<uint32_t>(n * per), static_cast<uint32_t>(std::min<int64_t>(cdiv(a.m - m0, MT * 16), 65535)));
    if (al)
      linear4_kernel<T, MT, RT, NW, true><<<grid, NW * 64, lds, s>>>(a);
    else
      linear4_kernel<T, MT, RT, NW, false><<<grid, NW * 64, lds, s>>>(a);
  }
}

template <typename T>
void dispatch(const Linear4& a, int64_t n, bool al, hipStream_t s) {
  if (a.m <= 16)
    launch<T, 1, 1, 4>(a, n, al, s);
  else if (a.m <= 32)
    launch<T, 2, 2, 4>(a, n, al, s);
  else
    launch<T, 4, 2, 4>(a, n, al, s);
}

}  // namespace
}  // namespace wc

extern "C" int32_t wc_linear4(const wc_linear4_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_linear4";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_linear4_args& p = *args;
  const int es = dtype_size(p.dtype);
  WC_REQUIRE(es, WC_ERR_DTYPE, "%s: dtype %d", what, p.dtype);
  WC_REQUIRE(p.group == 32 || p.group == 64 || p.group == 128, WC_ERR_ARG, "%s: group %d (32, 64 or 128)", what, p.group);
  WC_REQUIRE(p.n >= 0 && p.m >= 0 && p.o >= 0 && p.k >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(p.n < (1ll << 31) && p.m < (1ll << 31) - 128 && p.o < (1ll << 31) - 128 && p.k < (1ll << 30) &&
                 mul_sat({p.n, cdiv(p.o, 16)}) < (1ll << 22) && mul_sat({p.n, p.m, p.o, 4}) < INT64_MAX &&
                 mul_sat({p.n, p.o + 16, p.k + 128}) < INT64_MAX,
             WC_ERR_LIMIT, "%s: sizes beyond 32 bits, or more than 2^22 tiles of output rows", what);
  if (p.n == 0 || p.m == 0 || p.o == 0) return WC_OK;
  WC_REQUIRE(p.k > 0, WC_ERR_SHAPE, "%s: no columns", what);
  WC_REQUIRE(p.x && p.codes && p.scales && p.y, WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(p.x_rows_inner > 0, WC_ERR_ARG, "%s: rows_inner must be positive", what);
  WC_REQUIRE(p.x_rows_inner < (1ll << 31), WC_ERR_LIMIT, "%s: rows_inner beyond 32 bits", what);
  WC_REQUIRE(aligned(p.codes, 16) && aligned(p.scales, 16) && aligned(p.zeros, 4) && aligned(p.x, es) && aligned(p.y, es) &&
                 aligned(p.bias, es),
             WC_ERR_ALIGN, "%s: codes and scales must be 16-byte aligned, zeros 4-byte, the rest to their elements", what);
  Linear4 a;
  a.x = static_cast<const char*>(p.x);
  a.scales = static_cast<const char*>(p.scales);
  a.bias = static_cast<const char*>(p.bias);
  a.codes = static_cast<const uint8_t*>(p.codes);
  a.zeros = static_cast<const uint8_t*>(p.zeros);
  a.y = static_cast<char*>(p.y);
  a.xn = p.x_stride_n;
  a.xo = p.x_stride_outer;
  a.xi = p.x_stride_inner;
  a.m = static_cast<int32_t>(p.m);
  a.o = static_cast<int32_t>(p.o);
  a.k = static_cast<int32_t>(p.k);
  a.otiles = static_cast<int32_t>(cdiv(p.o, 16));
  a.ktiles = static_cast<int32_t>(cdiv(p.k, 128));
  a.steps_log2 = p.group == 32 ? 0 : p.group == 64 ? 1 : 2;
  a.by_rows = make_fastdiv(static_cast<uint32_t>(p.x_rows_inner));
  // whole vectors: of 8 columns in 16 bits, of 4 in fp32
  const bool al = p.k * es % 16 == 0 && aligned(p.x, 16) && ubytes(p.x_stride_n, es) % 16 == 0 &&
                  ubytes(p.x_stride_outer, es) % 16 == 0 && ubytes(p.x_stride_inner, es) % 16 == 0;
  const hipStream_t s = as_stream(stream);
  if (p.dtype == WC_F32)
    dispatch<float>(a, p.n, al, s);
  else if (p.dtype == WC_BF16)
    dispatch<bf16>(a, p.n, al, s);
  else
    dispatch<f16>(a, p.n, al, s);
  return check_launch(what);
}
