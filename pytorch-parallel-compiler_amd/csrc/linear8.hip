// Products in 8-bit integers: y = x W^T + bias with a scale for each row of x, found and applied here, and one for each
// output.
//
//   s = max(max |x| / 127, 2^-126),  c = round(x / s),   y[r, o] = s[r] scale[o] sum_k c[r, k] code[o, k] + bias[o]
//
// The sums are whole numbers in 32 bits (127^2 131072 < 2^31), so they are exact and no order of them matters: what a
// call gives depends on its row of x and on W alone.
//
// Both operands stand in tiles of 16 rows x 64 columns, in the order in which the lanes of v_mfma_i32_16x16x64_i8 take them: a
// tile is one kilobyte, loaded by a wave as it lies, into registers or by DMA into LDS, from where a lane reads its 16
// bytes at 16 times its number, without conflicts.  W is packed so once; x by the first of a call's two kernels.
#include <algorithm>

#include "wc_answer_abi.h"
#include "wc_codes.h"
#include "wc_linear8.h"

namespace wc {
namespace {

struct Linear8 {
  const char* x;
  const uint8_t* w;          // tiles [n][otiles][ktiles]
  uint8_t* c;                // tiles [n][mtiles][ktiles]
  float* s;                  // [n][mtiles * 16]
  const float* scales;
  const char* bias;
  char* y;
  int64_t xn, xo, xi;
  int32_t m, o, k, mtiles, otiles, ktiles;            // ktiles even
  FastDiv by_rows, by_mtiles, by_wg;                  // rows_inner; tiles of rows per model; workgroups per model
  int32_t vec;                                        // rows of y are whole vectors of four
};

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;

__device__ __forceinline__ i32x4 mma8(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// 16 values of a row, as they lie
template <typename T>
struct Piece {
  static constexpr int N = sizeof(T), E = 16 / sizeof(T);              // vectors, values of each
  u32x4 v[N];
  // those of lane group g in a tile, zeros from the row's end on
  __device__ __forceinline__ void load(const T* x, int tile, int g, int end) {
    const int k = tile * 64 + g * 16;
    if (tile * 64 + 64 <= end) {                      // the same for the wave
#pragma unroll
      for (int i = 0; i < N; ++i) __builtin_memcpy(&v[i], x + k + i * E, 16);          // at element alignment
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int at = k + i * E + q * (4 / static_cast<int>(sizeof(T)));
          uint32_t w = 0;
          if constexpr (sizeof(T) == 4) {
            if (at < end) w = __builtin_bit_cast(uint32_t, x[at]);
          } else {
            if (at < end) w = __builtin_bit_cast(uint16_t, x[at]);
            if (at + 1 < end) w |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, x[at + 1])) << 16;
          }
          v[i][q] = w;
        }
    }
  }
  __device__ __forceinline__ float value(int e) const {
    const uint32_t w = v[e / E][e % E / (4 / sizeof(T))];
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(float, w);
    else if constexpr (std::is_same<T, bf16>::value)
      return e & 1 ? bf16_hi(w) : bf16_lo(w);
    else
      return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(e & 1 ? w >> 16 : w)));
  }
  // the larger of `top` and the largest magnitude, as bits of the type: two 16-bit ones in a register, each of its own half
  __device__ __forceinline__ uint32_t top(uint32_t top) const {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t w = v[i][q];
        if constexpr (sizeof(T) == 4)
          top = std::max(top, w & 0x7fffffffu);
        else
          top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
      }
    return top;
  }
  // that as the bits of a float
  static __device__ __forceinline__ uint32_t as_float(uint32_t top) {
    if constexpr (sizeof(T) == 4)
      return top;
    else
      return __builtin_bit_cast(uint32_t, to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(std::max(top & 0xffffu, top >> 16)))));
  }
  static __device__ __forceinline__ u32x4 packed(const uint32_t (&code)[16], bool finite) {
    u32x4 o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t* c = code + 4 * q;
      const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
      o[q] = finite ? lo | hi << 16 : 0u;
    }
    return o;
  }
  __device__ __forceinline__ u32x4 codes(float scale, float inv, bool finite) const {
    uint32_t code[16];
    float far = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float off;
      code[e] = code8(value(e), scale, inv, off);
      far = fmaxf(far, off);
    }
    if (far > scale * kNearHalf)
#pragma unroll
      for (int e = 0; e < 16; ++e) code[e] = code8_near_half(value(e), scale, inv);
    return packed(code, finite);
  }
};

// What the sums of a row are multiplied by, whose largest magnitude as the bits of a float is `top`: its scale, NaN where it is not
// finite, and 1 where all is zero, as good there and a usual number
__device__ __forceinline__ float factor(uint32_t top) {
  return top >= 0x7f800000u ? __builtin_nanf("") : top == 0 ? 1.f : row_scale(top);
}

// Codes and scales of 16 rows of x: lane l has row l % 16 and columns 16 (l / 16).. of every tile of its wave, which is what
// it writes.  S workgroups share the codes of 16 rows, of which each looks for the scale by itself.  KEPT of its tiles a wave stay in
// registers until the scale is known; more are read a second time.  Memory and the three phases that all workgroups are in at
// once bound it: 2 x 4096 rows of 4096, 100 MB, 30 us (3.3 TB/s).
template <typename T, int NW, int KEPT, int S>
__global__ __launch_bounds__(NW * 64) void linear8_codes_kernel(Linear8 a) {
  __shared__ uint32_t tops[NW][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const uint32_t model = fdiv(blockIdx.x, a.by_mtiles);
  const int mt = blockIdx.x - model * a.by_mtiles.d;
  const uint32_t r = min(mt * 16 + j, a.m - 1), outer = fdiv(r, a.by_rows);        // past the last: the last again
  const T* x = reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (r - outer * a.by_rows.d) * a.xi;
  const int share = S == 1 ? 0 : blockIdx.y;
  auto own = [&](int i) { return (i * S + share) * NW + wave; };         // the workgroup's tiles, of the wave
  Piece<T> v[KEPT];
#pragma unroll
  for (int i = 0; i < KEPT; ++i) v[i].load(x, own(i), g, a.k);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < KEPT; ++i) top = v[i].top(top);
  // the others' and those behind the kept, four at a time on their way; past the last there are zeros
  if constexpr (S > 1) {
    const int others = (a.ktiles + NW * S - 1) / (NW * S) * (S - 1);
    for (int i0 = 0; i0 < others; i0 += 4) {
      Piece<T> u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e, round = i / (S - 1), s = i - round * (S - 1);
        u[e].load(x, (round * S + s + (s >= share)) * NW + wave, g, a.k);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) top = u[e].top(top);
    }
  }
  for (int i = KEPT; own(i) < a.ktiles; i += 4) {
    Piece<T> u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e].load(x, own(i + e), g, a.k);
#pragma unroll
    for (int e = 0; e < 4; ++e) top = u[e].top(top);
  }
  top = Piece<T>::as_float(top);
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
  if (g == 0) tops[wave][j] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) top = max(top, tops[w][j]);
  const bool finite = top < 0x7f800000u;
  const float scale = finite ? row_scale(top) : __builtin_nanf("");
  const float inv = __builtin_amdgcn_rcpf(scale);
  if (share == 0 && threadIdx.x < 16) a.s[static_cast<int64_t>(blockIdx.x) * 16 + j] = factor(top);
  u32x4* out = reinterpret_cast<u32x4*>(a.c) + static_cast<int64_t>(blockIdx.x) * a.ktiles * 64 + lane;
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
    if (own(i) < a.ktiles) out[static_cast<int64_t>(own(i)) * 64] = v[i].codes(scale, inv, finite);
#pragma unroll 1
  for (int i = KEPT; own(i) < a.ktiles; i += 4) {
    Piece<T> u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e].load(x, own(i + e), g, a.k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (own(i + e) < a.ktiles) out[static_cast<int64_t>(own(i + e)) * 64] = u[e].codes(scale, inv, finite);
  }
}

// Scales and bias of outputs o..o + 3
struct Columns {
  float scale[4], bias[4];
};
template <typename T>
__device__ __forceinline__ Columns columns(const Linear8& a, uint32_t model, int o) {
  Columns c;
  const int64_t at = static_cast<int64_t>(model) * a.o;
  const T* bias = reinterpret_cast<const T*>(a.bias);
  if (a.vec) {                                        // all four or none are there
    const int64_t i = at + (o < a.o ? o : 0);
    T b[4];
    __builtin_memcpy(c.scale, a.scales + i, 16);
    if (a.bias) __builtin_memcpy(b, bias + i, sizeof b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c.bias[e] = a.bias ? to_f32(b[e]) : 0.f;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t i = at + std::min(o + e, a.o - 1);
      c.scale[e] = a.scales[i];
      c.bias[e] = a.bias ? to_f32(bias[i]) : 0.f;
    }
  }
  return c;
}
__device__ __forceinline__ float row_of_scale(const Linear8& a, uint32_t model, int r) {
  return a.s[static_cast<int64_t>(model) * a.mtiles * 16 + std::min(r, a.m - 1)];
}
// Scales whose products with each other are normal numbers, whichever they are
__device__ __forceinline__ bool usual(float s) { return fabsf(s) >= 0x1p-63f && fabsf(s) <= 0x1p63f; }
__device__ __forceinline__ bool usual(const Columns& c) {
  bool all = true;
#pragma unroll
  for (int e = 0; e < 4; ++e) all &= usual(c.scale[e]) || c.scale[e] == 0.f;
  return all;
}
// sum s scale + bias where the scales' product may be too small or too large for fp32 though the result is not: what does not
// fit their product's exponent goes to the sum.
__device__ __forceinline__ float scaled_far(int sum, float s, float scale, float bias) {
  const int e = __builtin_amdgcn_frexp_expf(s) + __builtin_amdgcn_frexp_expf(scale), near = min(max(e, -120), 120);
  const float f = __builtin_amdgcn_ldexpf(__builtin_amdgcn_frexp_mantf(s) * __builtin_amdgcn_frexp_mantf(scale), near);
  return fmaf(__builtin_amdgcn_ldexpf(static_cast<float>(sum), e - near), f, bias);
}
// outputs o..o + 3 of row r, those there are; near: all scales of the wave are usual
template <typename T>
__device__ __forceinline__ void finish4(const Linear8& a, uint32_t model, int r, int o, i32x4 sum, float s, const Columns& c, bool near) {
  float f[4];
  if (near) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = static_cast<float>(sum[e]) * (s * c.scale[e]) + c.bias[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = scaled_far(sum[e], s, c.scale[e], c.bias[e]);
  }
  if (r >= a.m || o >= a.o) return;
  T* y = reinterpret_cast<T*>(a.y) + (static_cast<int64_t>(model) * a.m + r) * a.o + o;
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(f[e]);
  if (a.vec) {
    __builtin_memcpy(__builtin_assume_aligned(y, 4 * sizeof(T)), v, sizeof v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (o + e < a.o) y[e] = v[e];
  }
}
// a wave's FN x FM tiles
template <typename T, int FN, int FM>
__device__ __forceinline__ void finish(const Linear8& a, uint32_t model, int ot, int mt, int lane, const i32x4 (&acc)[FN][FM]) {
  float s[FM];
  bool rows = true;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    s[j] = row_of_scale(a, model, (mt + j) * 16 + (lane & 15));
    rows &= usual(s[j]);
  }
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int o = (ot + i) * 16 + (lane >> 4) * 4;
    const Columns c = columns<T>(a, model, o);
    const bool near = __all(rows && usual(c));
#pragma unroll
    for (int j = 0; j < FM; ++j) finish4<T>(a, model, (mt + j) * 16 + (lane & 15), o, acc[i][j], s[j], c, near);
  }
}
// a barrier that waits for nothing but the other waves
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Up to 16 rows of x a workgroup: it has RT tiles of output rows, its waves every NW-th tile of columns, D of them on their way.
// W bounds it, read once from memory without LDS.
template <typename T, int RT, int NW, int D>
__global__ __launch_bounds__(NW * 64) void linear8_few_kernel(Linear8 a) {
  __shared__ i32x4 part[NW][RT][64];
  // the wave's number as a scalar: matrix instructions take no notice of lanes that a condition has switched off
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t model = fdiv(blockIdx.x, a.by_wg);
  const int ot0 = (blockIdx.x - model * a.by_wg.d) * RT, mt = blockIdx.y;
  const i32x4* x = reinterpret_cast<const i32x4*>(a.c) + (static_cast<int64_t>(model) * a.mtiles + mt) * a.ktiles * 64 + lane;
  const i32x4* w[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
    w[t] = reinterpret_cast<const i32x4*>(a.w) + (static_cast<int64_t>(model) * a.otiles + min(ot0 + t, a.otiles - 1)) * a.ktiles * 64 + lane;
  i32x4 acc[RT] = {}, wf[D][RT], xf[D];
  auto fetch = [&](int d, int kt) {                   // past the last: the last again
    const int64_t at = static_cast<int64_t>(min(kt, a.ktiles - 1)) * 64;
#pragma unroll
    for (int t = 0; t < RT; ++t) wf[d][t] = w[t][at];
    xf[d] = x[at];
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(d, wave + d * NW);
  for (int k0 = wave; k0 < a.ktiles; k0 += D * NW) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (k0 + d * NW < a.ktiles)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t] = mma8(wf[d][t], xf[d], acc[t]);
      fetch(d, k0 + (d + D) * NW);
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  // lane: outputs 4 (lane / 16).. of row lane % 16
  for (int t = wave; t < RT; t += NW) {
    i32x4 sum = part[0][t][lane];
#pragma unroll
    for (int v = 1; v < NW; ++v) sum += part[v][t][lane];
    const int r = mt * 16 + (lane & 15), o = (ot0 + t) * 16 + (lane >> 4) * 4;
    const float scale = row_of_scale(a, model, r);
    const Columns c = columns<T>(a, model, o);
    finish4<T>(a, model, r, o, sum, scale, c, __all(usual(scale) && usual(c)));
  }
}

// The same for so few rows of x (kFusedPieces pieces of 16 columns in all) that every workgroup finds their codes for itself,
// in LDS, while its first weights are on their way: a launch costs more (four models' [4096 -> 4096], one row: 13.7 us, 4.9 TB/s; with
// a launch for the codes 21.0; four rows 16.9 and 23.2).
template <typename T, int RT, int NW, int D>
__global__ __launch_bounds__(NW * 64) void linear8_fused_kernel(Linear8 a) {
  constexpr int NT = NW * 64, KEPT = kFusedPieces / NT;
  __shared__ i32x4 part[NW][RT][64];
  __shared__ u32x4 codes[kFusedPieces];              // [row][columns / 16]
  __shared__ uint32_t tops[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, g = lane >> 4;
  const uint32_t model = fdiv(blockIdx.x, a.by_wg);
  const int ot0 = (blockIdx.x - model * a.by_wg.d) * RT;
  const i32x4* w[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
    w[t] = reinterpret_cast<const i32x4*>(a.w) + (static_cast<int64_t>(model) * a.otiles + min(ot0 + t, a.otiles - 1)) * a.ktiles * 64 + lane;
  // piece tid + i NT of x: row p / (4 ktiles), columns 16 (p % (4 ktiles))..
  const int per = a.ktiles * 4, pieces = a.m * per;
  Piece<T> v[KEPT];
  int row[KEPT];
#pragma unroll
  for (int i = 0; i < KEPT; ++i) {
    const int p = min(tid + i * NT, pieces - 1), c = p % per;
    row[i] = p / per;
    const uint32_t outer = fdiv(row[i], a.by_rows);
    v[i].load(reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (row[i] - outer * a.by_rows.d) * a.xi, c >> 2, c & 3, a.k);
  }
  i32x4 acc[RT] = {}, wf[D][RT];
  auto fetch = [&](int d, int kt) {                   // past the last: the last again
    const int64_t at = static_cast<int64_t>(min(kt, a.ktiles - 1)) * 64;
#pragma unroll
    for (int t = 0; t < RT; ++t) wf[d][t] = w[t][at];
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(d, wave + d * NW);
  if (tid < 16) tops[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < KEPT; ++i) {
    uint32_t top = Piece<T>::as_float(v[i].top(0));
    if (__all(row[i] == __builtin_amdgcn_readfirstlane(row[i]))) {
#pragma unroll
      for (int off = 32; off; off >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 64)));
      if (lane == 0) atomicMax(&tops[row[i]], top);
    } else {
      atomicMax(&tops[row[i]], top);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < KEPT; ++i) {
    if (tid + i * NT >= pieces) continue;
    const uint32_t top = tops[row[i]];
    const bool finite = top < 0x7f800000u;
    const float scale = finite ? row_scale(top) : __builtin_nanf("");
    codes[tid + i * NT] = v[i].codes(scale, __builtin_amdgcn_rcpf(scale), finite);
  }
  __syncthreads();
  const u32x4* mine = codes + min(j, a.m - 1) * per + g;
#pragma unroll 1
  for (int k0 = wave; k0 < a.ktiles; k0 += D * NW) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int kt = k0 + d * NW;
      if (kt < a.ktiles) {
        const i32x4 c = __builtin_bit_cast(i32x4, mine[kt * 4]);       // lanes without a row have another's
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t] = mma8(wf[d][t], c, acc[t]);
      }
      fetch(d, kt + D * NW);
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < RT; t += NW) {
    i32x4 sum = part[0][t][lane];
#pragma unroll
    for (int e = 1; e < NW; ++e) sum += part[e][t][lane];
    const uint32_t top = tops[min(j, a.m - 1)];
    const int o = (ot0 + t) * 16 + g * 4;
    const float scale = factor(top);
    const Columns c = columns<T>(a, model, o);
    finish4<T>(a, model, j, o, sum, scale, c, __all(usual(scale) && usual(c)));
  }
}

// Tiles of BM x BN outputs through LDS: WM x WN waves of FM x FN tiles each, NS stages of 128 columns in a ring, brought by DMA.  Eight
// models' 64 rows [2048 -> 8192], 143 MB: 36.6 us with weights from memory (3.9 TB/s), 29.7 with those that a call before left in the
// cache; accumulators stand in AGPRs and are copied in every stage.
template <typename T, int FM, int FN, int WM, int WN, int NS>
__global__ __launch_bounds__(WM * WN * 64) void linear8_tile_kernel(Linear8 a) {
  constexpr int NW = WM * WN, TM = FM * WM, TN = FN * WN, PIECES = (TM + TN) * 2, PER = PIECES / NW;
  static_assert(PIECES % NW == 0, "every wave brings as many pieces");
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];       // [NS][TN + TM][2] tiles
  lds_char* const lds = (lds_char*)lds_raw;            // keeps every LDS address 32-bit
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t model = fdiv(blockIdx.x, a.by_wg), rem = blockIdx.x - model * a.by_wg.d;
  const int per = (a.mtiles + TM - 1) / TM, ot0 = rem / per * TN, mt0 = rem % per * TM;
  // piece p of a stage: half p % 2 of tile p / 2, those of W first; tiles past the last are the last again
  const uint8_t* src[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int p = wave * PER + i, t = p >> 1;
    const int64_t row = t < TN ? static_cast<int64_t>(model) * a.otiles + min(ot0 + t, a.otiles - 1)
                               : static_cast<int64_t>(model) * a.mtiles + min(mt0 + t - TN, a.mtiles - 1);
    src[i] = (t < TN ? a.w : a.c) + (row * a.ktiles + (p & 1)) * 1024 + lane * 16;
  }
  const int stages = a.ktiles / 2;
  auto issue = [&](int s) {                            // past the last: the last again, which keeps the count of loads
    const int64_t at = static_cast<int64_t>(min(s, stages - 1)) * 2048;
    lds_char* const to = lds + (s % NS) * (PIECES * 1024) + wave * PER * 1024;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const void*>(src[i] + at), (lds_ptr_t)(to + i * 1024), 16, 0, 0);
  };
  i32x4 acc[FN][FM] = {};
  const int wm = wave / WN * FM, wn = wave % WN * FN;
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(s);
  for (int s = 0; s < stages; ++s) {
    // stage s has landed for this wave, then for all; the slot of stage s - 1 is free
    __builtin_amdgcn_s_waitcnt((((NS - 2) * PER) & 15) | ((((NS - 2) * PER) >> 4) << 14) | 0x0070 | 0x0f00);
    bare_barrier();
    issue(s + NS - 1);
    const lds_char* const st = lds + (s % NS) * (PIECES * 1024) + lane * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 wf[FN], xf[FM];
#pragma unroll
      for (int i = 0; i < FN; ++i) wf[i] = *(const lds_i32x4*)(st + ((wn + i) * 2 + h) * 1024);
#pragma unroll
      for (int j = 0; j < FM; ++j) xf[j] = *(const lds_i32x4*)(st + ((TN + wm + j) * 2 + h) * 1024);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = mma8(wf[i], xf[j], acc[i][j]);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);                  // no DMA outlives the workgroup
  finish<T>(a, model, ot0 + wn, mt0 + wm, lane, acc);
}

// Tiles of 256 x 256 outputs for whole rounds of the compute units: 8 waves of 128 outputs x 64 rows each, four stages of 64 columns
// in LDS.  A workgroup walks its tiles without a pause between them: stages of all its tiles are one line, and while one is
// multiplied the next three are on their way.  Within a stage the waves stream their tiles of W through four registers,
// four groups of MFMAs ahead of their use, so that a wave seldom waits for what it reads.  Two models' 4096 rows [4096 -> 4096]: 128 us,
// 2.1e15 operations a second.  LDS bounds it: a stage is 1024 cycles of MFMAs, and as many to write its 32 KB and read 96 KB out of
// it at 128 bytes a cycle.  (Two stages of 128 columns took 137 us; four waves of 128 x 128, which read a third less, 161 us, as
// one wave a SIMD hides nothing and 256 accumulators leave too few registers.)
constexpr int kLargeThreads = 512, kLargeStage = 2 * kLargeTiles * 1024;

template <typename T>
__global__ __launch_bounds__(kLargeThreads, 1) void linear8_large_kernel(Linear8 a, int tiles_total, int per) {
  __shared__ __attribute__((aligned(1024))) char raw[4 * kLargeStage];       // [4][W tiles, x tiles]
  lds_char* const lds = (lds_char*)raw;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = (wave & 1) * 8, wm = (wave >> 1) * 4, stages = a.ktiles;
  // this workgroup's tiles: XCD x = blockIdx % 8 has a range of neighbours, which share what they read
  const int grid = gridDim.x;
  int first = blockIdx.x, step = grid, mine;
  if (grid % 8 == 0) {
    const int x = blockIdx.x & 7, lo = static_cast<int>(static_cast<int64_t>(tiles_total) * x >> 3);
    const int hi = static_cast<int>(static_cast<int64_t>(tiles_total) * (x + 1) >> 3);
    step = grid >> 3;
    first = lo + (blockIdx.x >> 3);
    mine = first < hi ? (hi - first + step - 1) / step : 0;
  } else {
    mine = first < tiles_total ? (tiles_total - first + step - 1) / step : 0;
  }
  if (mine == 0) return;
  struct Tile {
    uint32_t model;
    int ot, mt;
  };
  auto tile_of = [&](int i) {
    // neighbours are 8 tiles along the rows by 4 along the outputs: 32 compute units of an XCD read 12 tiles' operands
    const uint32_t t = first + i * step, model = fdiv(t, a.by_wg), rem = t - model * a.by_wg.d;
    const int ots = a.by_wg.d / per, band = rem / (8 * ots), high = std::min(8, per - band * 8), in = rem - band * 8 * ots;
    return Tile{model, in / high * kLargeTiles, (band * 8 + in % high) * kLargeTiles};
  };
  // What comes next: tiles 2 wave and 2 wave + 1 of W, then of x; past the last stage the last again, which keeps the count of loads.
  const uint8_t* from[4];
  int coming = 0, left = 0, to = 0;                    // tile, its stages that are left, slot
  auto aim = [&](int i) {
    const Tile t = tile_of(i);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      from[e] = a.w + (static_cast<int64_t>(t.model) * a.otiles + std::min(t.ot + 2 * wave + e, a.otiles - 1)) * a.ktiles * 1024;
      from[2 + e] = a.c + (static_cast<int64_t>(t.model) * a.mtiles + std::min(t.mt + 2 * wave + e, a.mtiles - 1)) * a.ktiles * 1024;
    }
    coming = i;
    left = stages;
  };
  auto bring = [&](int q) __attribute__((always_inline)) {
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const void*>(from[q] + lane * 16),
                                     (lds_ptr_t)(lds + to * kLargeStage + (q >> 1) * (kLargeStage / 2) + (2 * wave + (q & 1)) * 1024), 16, 0, 0);
  };
  auto next = [&]() __attribute__((always_inline)) {
    to = (to + 1) & 3;
    if (left > 1) {
      --left;
#pragma unroll
      for (int e = 0; e < 4; ++e) from[e] += 1024;
    } else if (coming + 1 < mine) {
      aim(coming + 1);
    }
  };
  i32x4 acc[8][4], wr[4], xa[4], xb[4];
  auto read_w = [&](int slot, int g) __attribute__((always_inline)) {
    wr[g & 3] = *(const lds_i32x4*)(lds + slot * kLargeStage + (wn + g) * 1024 + lane * 16);
  };
  auto read_x = [&](int slot, i32x4(&x)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = *(const lds_i32x4*)(lds + slot * kLargeStage + kLargeStage / 2 + (wm + j) * 1024 + lane * 16);
  };
  aim(0);
#pragma unroll
  for (int s = 0; s < 3; ++s) {
#pragma unroll
    for (int q = 0; q < 4; ++q) bring(q);
    next();
  }
  bring(0);
  bring(1);
  __builtin_amdgcn_s_waitcnt(0x0070 | 10);             // of 14 loads the first stage's
  bare_barrier();
#pragma unroll
  for (int g = 0; g < 4; ++g) read_w(0, g);
  read_x(0, xa);
  // the stage in a slot; its rows of x are in x, those of the next come into y
  auto stage = [&](int slot, const i32x4(&x)[4], i32x4(&y)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 8; ++g) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[g][j] = mma8(wr[g & 3], x[j], acc[g][j]);
        if (j == 1 && (g < 2 || g > 5)) {              // one load at a time: back to back they stall the wave
          __builtin_amdgcn_sched_barrier(0);
          bring(g < 2 ? 2 + g : g - 6);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (g == 1) next();
      if (g + 4 < 8) read_w(slot, g + 4);
      if (g == 5) {
        // the wave's reads of this stage are done and the next has landed, which leaves two stages of four loads on their way; then
        // all waves': the slot can take the next but three
        __builtin_amdgcn_s_waitcnt(0x0070 | 8);
        bare_barrier();
        read_x((slot + 1) & 3, y);
        read_w((slot + 1) & 3, 0);
        read_w((slot + 1) & 3, 1);
      }
      if (g == 6) read_w((slot + 1) & 3, 2);
      if (g == 7) read_w((slot + 1) & 3, 3);
    }
  };
  int slot = 0;
  for (int i = 0; i < mine; ++i) {
#pragma unroll
    for (int g = 0; g < 8; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[g][j] = i32x4{0, 0, 0, 0};
    for (int k = 0; k < stages; k += 2) {              // of whole tiles of 128 columns
      stage(slot, xa, xb);
      stage(slot + 1, xb, xa);
      slot = (slot + 2) & 3;
    }
    const Tile t = tile_of(i);
    finish<T>(a, t.model, t.ot + wn, t.mt + wm, lane, acc);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);                  // no DMA outlives the workgroup
}

template <typename T, int RT, int NW, int D>
void launch_few(Linear8 a, int64_t n, hipStream_t s) {
  const int64_t per = cdiv(a.otiles, RT);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(per));
  linear8_few_kernel<T, RT, NW, D><<<dim3(static_cast<uint32_t>(n * per), static_cast<uint32_t>(a.mtiles)), NW * 64, 0, s>>>(a);
}

template <typename T, int RT, int NW, int D>
void launch_fused(Linear8 a, int64_t n, hipStream_t s) {
  const int64_t per = cdiv(a.otiles, RT);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(per));
  linear8_fused_kernel<T, RT, NW, D><<<static_cast<uint32_t>(n * per), NW * 64, 0, s>>>(a);
}

template <typename T, int FM, int FN, int WM, int WN, int NS>
void launch_tile(Linear8 a, int64_t n, hipStream_t s) {
  const int64_t per = cdiv(a.mtiles, FM * WM) * cdiv(a.otiles, FN * WN);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(per));
  const size_t lds = static_cast<size_t>(NS) * (FM * WM + FN * WN) * 2048;
  const auto kernel = linear8_tile_kernel<T, FM, FN, WM, WN, NS>;
  if (lds > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
  kernel<<<static_cast<uint32_t>(n * per), WM * WN * 64, lds, s>>>(a);
}

template <typename T>
void launch_large(Linear8 a, int64_t n, hipStream_t s) {
  const int64_t per = cdiv(a.mtiles, kLargeTiles), tiles = per * cdiv(a.otiles, kLargeTiles);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(tiles));
  const int64_t grid = std::min<int64_t>(n * tiles, std::max(device_cu_count(), 8));
  linear8_large_kernel<T><<<static_cast<uint32_t>(grid), kLargeThreads, 0, s>>>(a, static_cast<int>(n * tiles), static_cast<int>(per));
}

template <typename T>
void launch(const Linear8& a, int64_t n, hipStream_t s) {
  const uint32_t tiles = static_cast<uint32_t>(n * a.mtiles);
  const Linear8Form form = linear8_form(n, a.m, a.mtiles, a.otiles, a.ktiles);
  if (form == Linear8Form::fused) return launch_fused<T, 1, 4, 8>(a, n, s);
  // Where rows' tiles are fewer than compute units, more waves have them (256 rows [1024 -> 1024], eight models: by four waves 21.8 us for
  // the whole product, by 16 18.0), and of longer rows four workgroups, each with a quarter of the codes (64 rows [4096 -> 4096]: by
  // one of eight waves 26.0, by four 19.7; 129 rows [7280 -> 416], two models: 29.9 and 23.4).
  if (tiles < 256 && a.ktiles <= 16)
    linear8_codes_kernel<T, 16, 1, 1><<<tiles, 1024, 0, s>>>(a);
  else if (tiles < 256 && a.ktiles <= 32)
    linear8_codes_kernel<T, 8, 1, 4><<<dim3(tiles, 4), 512, 0, s>>>(a);
  else if (tiles < 256)
    linear8_codes_kernel<T, 8, 4, 4><<<dim3(tiles, 4), 512, 0, s>>>(a);
  else if (a.ktiles <= 16)
    linear8_codes_kernel<T, 4, 4, 1><<<tiles, 256, 0, s>>>(a);
  else if (a.ktiles <= 64 || sizeof(T) == 4)
    linear8_codes_kernel<T, 8, 8, 1><<<tiles, 512, 0, s>>>(a);
  else if constexpr (sizeof(T) != 4)
    linear8_codes_kernel<T, 16, 8, 1><<<tiles, 1024, 0, s>>>(a);
  switch (form) {
    case Linear8Form::few: return launch_few<T, 1, 4, 8>(a, n, s);
    case Linear8Form::ring6: return launch_tile<T, 4, 2, 1, 4, 6>(a, n, s);
    case Linear8Form::ring3: return launch_tile<T, 4, 2, 1, 4, 3>(a, n, s);
    case Linear8Form::large: return launch_large<T>(a, n, s);
    default: return launch_tile<T, 4, 4, 2, 2, 2>(a, n, s);
  }
}

int32_t check(const wc_linear8_args& p, const char* what) {
  WC_REQUIRE(dtype_size(p.dtype), WC_ERR_DTYPE, "%s: dtype %d", what, p.dtype);
  WC_REQUIRE(p.n >= 0 && p.m >= 0 && p.o >= 0 && p.k >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(p.k <= 131072, WC_ERR_LIMIT, "%s: %lld columns, whose sums could pass 32 bits (at most 131072)", what, (long long)p.k);
  // tiles are counted in 32 bits, bytes in 64
  WC_REQUIRE(p.m < (1ll << 31) - 1024 && p.o < (1ll << 31) - 1024 && p.n < (1ll << 31) &&
                 mul_sat({p.n, cdiv(p.m, 16)}) < (1ll << 22) && mul_sat({p.n, cdiv(p.o, 16)}) < (1ll << 22) &&
                 mul_sat({p.n, cdiv(p.m, 16), cdiv(p.o, 16)}) < (1ll << 29),
             WC_ERR_LIMIT, "%s: more than 2^22 tiles of 16 rows or of 16 outputs, or 2^29 of both", what);
  return WC_OK;
}

// codes, then scales
int64_t code_bytes(const wc_linear8_args& p) { return p.n * cdiv(p.m, 16) * cdiv(p.k, 128) * 2048; }
int64_t workspace_of(const wc_linear8_args& p) { return code_bytes(p) + p.n * cdiv(p.m, 16) * 64; }
bool nothing(const wc_linear8_args& p) { return p.n == 0 || p.m == 0 || p.o == 0; }

}  // namespace
}  // namespace wc

extern "C" int64_t wc_linear8_workspace_bytes(const wc_linear8_args* args) {
  using namespace wc;
  clear_error();
  if (!args) {
    set_error(WC_ERR_NULL, "wc_linear8: null args");
    return -1;
  }
  if (check(*args, "wc_linear8")) return -1;
  return nothing(*args) ? 0 : workspace_of(*args);
}

extern "C" int32_t wc_linear8(const wc_linear8_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_linear8";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_linear8_args& p = *args;
  if (int32_t rc = check(p, what)) return rc;
  if (nothing(p)) return WC_OK;
  const int es = dtype_size(p.dtype);
  WC_REQUIRE(p.k > 0, WC_ERR_SHAPE, "%s: no columns", what);
  WC_REQUIRE(p.x && p.codes && p.scales && p.y, WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(p.x_rows_inner > 0, WC_ERR_ARG, "%s: rows_inner must be positive", what);
  WC_REQUIRE(p.x_rows_inner < (1ll << 31), WC_ERR_LIMIT, "%s: rows_inner beyond 32 bits", what);
  WC_REQUIRE(aligned(p.codes, 16) && aligned(p.scales, 4) && aligned(p.x, es) && aligned(p.y, es) && aligned(p.bias, es),
             WC_ERR_ALIGN, "%s: codes must be 16-byte aligned, the rest to their elements", what);
  const int64_t need = workspace_of(p);
  WC_REQUIRE(p.workspace && p.workspace_bytes >= need, WC_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what,
             (long long)p.workspace_bytes, (long long)need);
  WC_REQUIRE(aligned(p.workspace, 16), WC_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  Linear8 a;
  a.x = static_cast<const char*>(p.x);
  a.w = static_cast<const uint8_t*>(p.codes);
  a.c = static_cast<uint8_t*>(p.workspace);
  a.s = reinterpret_cast<float*>(a.c + code_bytes(p));
  a.scales = p.scales;
  a.bias = static_cast<const char*>(p.bias);
  a.y = static_cast<char*>(p.y);
  a.xn = p.x_stride_n;
  a.xo = p.x_stride_outer;
  a.xi = p.x_stride_inner;
  a.m = static_cast<int32_t>(p.m);
  a.o = static_cast<int32_t>(p.o);
  a.k = static_cast<int32_t>(p.k);
  a.mtiles = static_cast<int32_t>(cdiv(p.m, 16));
  a.otiles = static_cast<int32_t>(cdiv(p.o, 16));
  a.ktiles = static_cast<int32_t>(cdiv(p.k, 128)) * 2;
  a.by_rows = make_fastdiv(static_cast<uint32_t>(p.x_rows_inner));
  a.by_mtiles = make_fastdiv(static_cast<uint32_t>(a.mtiles));
  a.vec = p.o % 4 == 0 && aligned(p.y, 4 * es);
  const hipStream_t s = as_stream(stream);
  if (p.dtype == WC_F32)
    launch<float>(a, p.n, s);
  else if (p.dtype == WC_BF16)
    launch<bf16>(a, p.n, s);
  else
    launch<f16>(a, p.n, s);
  return check_launch(what);
}

extern "C" int32_t wc_answer_abi_version(void) { return WC_ANSWER_ABI_VERSION; }
