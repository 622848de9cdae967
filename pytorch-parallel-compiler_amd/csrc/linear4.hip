// Products with weights of 4 bits: y = x W^T + bias, W[o, k] = scale[o, g] (code[o, k] - zero[o, g]), g = k / group.
//
// For the few rows of x that answering token by token has, the weights' bytes bound it: half a byte a weight against
// 2 flops a row.  So the weights are read once, as whole kilobytes per wave (a tile of 16 output rows x 128 columns
// is laid out in the order in which the lanes want it), and all rows of x meet them there, 16 to an MFMA tile.
//
//   y = sum_g scale_g sum_k (code - zero_g) x
//
// A code less its zero point is a whole number that bf16 and fp16 hold, so what enters the product is exact, a weight of 0
// takes no part however large x is there, and the scale multiplies the fp32 sum of each group.  fp16: 0x6400 | code is
// 1024 + code, two to an instruction, and 1024 + zero is taken off two at a time.  bf16 has no packed subtraction: four
// codes a register lose their zero points as bytes, and each becomes a float and one half of a bf16 pair.  (Numbers
// 128 + code, with 128 + zero times the sum of x taken off afterwards, are half the instructions for the codes, but as many
// more for those sums: 4 models' [4096 -> 4096], one row, 11.8 us against 12.6, 8 models' [2048 -> 8192], 64 rows, 47 against
// 42, weights from memory; and they lose 2^-24 of 143 sum |x|, also where weights are 0, and overflow from x of 2^114 on.)
// fp32 goes as three bf16 planes of x (every bit of it down to 2^-110); a row of x with an infinity gives NaN there.
//
// 4 models' [4096 -> 4096] in bf16, one row (35 MB): 11.1 us, of which an empty launch is 3.3; 8 models' [2048 -> 8192]
// in fp16, 64 rows (84 MB, 17 GFLOP): 30 us, half of it the instructions that make numbers of codes and scale the
// groups' sums, which with two to four waves a unit's quarter only partly hide behind the loads.
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
  int32_t m, o, k, otiles, ktiles, m0;                // m0: first row of x of a launch
  int32_t vec;                                        // rows of x are whole 16-byte vectors
  FastDiv by_rows, by_wg;                             // rows_inner; workgroups per model
};

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

// 8 codes of a word less their zero point, as bf16 (fp32 too) or fp16.  `zero`: the zero point in each byte (bf16) or 1024
// and it in each half (fp16); `over`: the bits that stand above a code meanwhile, in a register, so that mask and bits are
// one instruction.  bf16: a byte 128 + code takes a zero point of up to 127 off without borrowing, then its top bit is the
// sign's again, and a signed byte becomes a float in one instruction.
template <typename T>
__device__ __forceinline__ u32x4 numbers(uint32_t w, uint32_t zero, uint32_t over) {
  u32x4 r;
  if constexpr (std::is_same<T, f16>::value) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, ((w >> (4 * e)) & 0x000f000fu) | over) - __builtin_bit_cast(h2, zero));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t v = ((((w >> (4 * (e & 1))) & 0x0f0f0f0fu) | over) - zero) ^ over;
      r[e] = pack_bf16x2(byte_f32(v, e / 2), byte_f32(v, e / 2 + 2));
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t bits_over() {
  uint32_t v;
  if constexpr (std::is_same<T, f16>::value)
    asm("v_mov_b32 %0, 0x64006400" : "=v"(v));
  else
    asm("v_mov_b32 %0, 0x80808080" : "=v"(v));
  return v;
}
template <typename T>
__device__ __forceinline__ uint32_t zero_point(uint32_t z) {
  return std::is_same<T, f16>::value ? __builtin_amdgcn_perm(0u, z, 0x01000100u) + 0x64006400u : __builtin_amdgcn_perm(0u, z, 0u);
}

// A tile of weights in a lane's registers: codes of row j and, for each of the GP groups of its 128 columns, that row's zero
// point, and the scales of rows 4 g + 0..3, whose sums the lane has
template <typename T, int GP>
struct Tile {
  u32x4 w;
  Four<T> scale[GP];
  uint32_t zero[GP];
};
template <typename T, int GP>
struct TileSource {
  const u32x4* codes;
  const T* scales;
  const uint8_t* zeros;
  int last;
  __device__ __forceinline__ TileSource(const Linear4& a, uint32_t model, int ot, int lane) {
    const int64_t t = static_cast<int64_t>(model) * a.otiles + std::min(ot, a.otiles - 1);
    codes = reinterpret_cast<const u32x4*>(a.codes) + t * a.ktiles * 64 + lane;
    scales = reinterpret_cast<const T*>(a.scales) + t * a.ktiles * (GP * 16) + (lane >> 4) * 4;
    zeros = a.zeros + t * a.ktiles * (GP * 16) + (lane & 15);
    last = a.ktiles - 1;
  }
  __device__ __forceinline__ void load(Tile<T, GP>& t, int kt) const {      // past the last: the last again
    const int k = std::min(kt, last);
    t.w = codes[k * 64];
#pragma unroll
    for (int s = 0; s < GP; ++s) {
      const int64_t m = static_cast<int64_t>(k) * GP * 16 + s * 16;
      t.scale[s] = *reinterpret_cast<const Four<T>*>(scales + m);
      t.zero[s] = zeros[m];
    }
  }
};

// acc += RT tiles of weights times MT * 16 rows of x; x(q, xf): the planes of all rows of columns 32 q..
template <typename T, int GP, int RT, int MT, typename X>
__device__ __forceinline__ void multiply(const Tile<T, GP> (&tile)[RT], uint32_t over, X x, f32x4 (&acc)[RT][MT]) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int NX = kF32 ? 3 : 1, STEPS = 4 / GP;
  typedef typename std::conditional<std::is_same<T, f16>::value, f16, bf16>::type MM;
#pragma unroll
  for (int s = 0; s < GP; ++s) {
    f32x4 part[RT][MT] = {};
#pragma unroll
    for (int q = s * STEPS; q < (s + 1) * STEPS; ++q) {
      u32x4 xf[MT][NX];
      x(q, xf);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const u32x4 c = numbers<T>(tile[r].w[q], zero_point<T>(tile[r].zero[s]), over);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = NX - 1; n >= 0; --n)
            part[r][t] = mma16<MM>(__builtin_bit_cast(bf16x8, c), __builtin_bit_cast(bf16x8, xf[t][n]), part[r][t]);
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float scale = to_f32(tile[r].scale[s].v[e]);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t][e] += scale * part[r][t][e];
      }
  }
}

__device__ __forceinline__ bool aligned_device(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T>
__device__ __forceinline__ const T* x_row(const Linear4& a, uint32_t model, int row) {
  const uint32_t r = std::min(row, a.m - 1), outer = fdiv(r, a.by_rows);    // past the last: the last again
  return reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (r - outer * a.by_rows.d) * a.xi;
}

// 16 bytes of a row of x at column k, and its values from the row's end on as zeros: apart, because what looks at a
// loaded value waits for it.  Rows that aren't whole vectors (AL false) are loaded at any address all the same, the piece
// over the end from further left, and moved down afterwards; value by value only where a row is shorter than a vector.
template <typename T, bool AL>
__device__ __forceinline__ u32x4 x_load(const T* x, int k, int end) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (AL) return *reinterpret_cast<const u32x4*>(x + (k < end ? k : 0));
  u32x4 v;
  if (end >= E) {
    __builtin_memcpy(&v, x + std::min(k, end - E), sizeof v);
  } else {
    T s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = x[k + e < end ? k + e : 0];
    __builtin_memcpy(&v, s, sizeof v);
  }
  return v;
}
template <typename T, bool AL>
__device__ __forceinline__ u32x4 x_keep(u32x4 v, int k, int end) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (AL) return k < end ? v : u32x4{};
  if (end >= E) {
    const int down = std::max(k - (end - E), 0) * static_cast<int>(sizeof(T)) * 8;      // bits
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    const u64x2 w = __builtin_bit_cast(u64x2, v);
    const u64x2 part = down < 64 ? u64x2{w[0] >> (down & 63) | w[1] << 1 << (~down & 63), w[1] >> (down & 63)} : u64x2{w[1] >> (down & 63), 0};
    return down == 0 ? v : down < 128 ? __builtin_bit_cast(u32x4, part) : u32x4{};
  }
  T s[E];
  __builtin_memcpy(s, &v, sizeof v);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (k + e >= end) s[e] = static_cast<T>(0.f);
  __builtin_memcpy(&v, s, sizeof v);
  return v;
}

// outputs o..o + 3 of a row of y, those it has
template <typename T>
__device__ __forceinline__ void store4(T* y, int o, int end, const T* bias, f32x4 s) {
  Four<T> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (bias && o + e < end) s[e] += to_f32(bias[o + e]);
    r.v[e] = from_f32<T>(s[e]);
  }
  if (o + 4 <= end && aligned_device(y + o, sizeof(r)))
    *reinterpret_cast<Four<T>*>(y + o) = r;
  else
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (o + e < end) y[o + e] = r.v[e];
}

// Up to 16 rows of x, straight from memory: a workgroup has RT tiles of output rows, its waves every NW-th tile of
// columns.  Weights come D tiles ahead of their use, x (which all workgroups share, in L2) one.
template <typename T, int GP, int RT, int NW, bool AL>
__global__ __launch_bounds__(NW * 64) void linear4_few_kernel(Linear4 a) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int NX = kF32 ? 3 : 1, D = RT * GP > 4 || (RT > 1 && (kF32 || NW > 4)) ? 2 : 4, E = 16 / sizeof(T), P = 8 / E;
  __shared__ float lds[NW * 16 * RT * 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const uint32_t model = fdiv(blockIdx.x, a.by_wg);
  const int ot = (blockIdx.x - model * a.by_wg.d) * RT;
  const int row0 = a.m0 + blockIdx.y * 16;
  const T* x = x_row<T>(a, model, row0 + j);
  const uint32_t over = bits_over<T>();

  struct Columns {
    u32x4 v[4][P];                       // 8 columns of each 32
  };
  auto bring = [&](Columns& c, int kt) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int h = 0; h < P; ++h) c.v[q][h] = x_load<T, AL>(x, kt * 128 + q * 32 + g * 8 + h * E, a.k);
  };

  f32x4 acc[RT][1] = {};
  Tile<T, GP> tile[D][RT];
  auto fetch = [&](int slot, int kt) {
#pragma unroll
    for (int t = 0; t < RT; ++t) TileSource<T, GP>(a, model, ot + t, lane).load(tile[slot][t], kt);
  };
  Columns cols[2];
#pragma unroll
  for (int i = 0; i < D; ++i) fetch(i, wave + i * NW);
  bring(cols[0], wave);
  for (int kt0 = wave; kt0 < a.ktiles; kt0 += D * NW) {
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const int kt = kt0 + i * NW;
      if (kt < a.ktiles) {
        bring(cols[(i + 1) & 1], kt + NW);
        u32x4 xf[4][NX];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          u32x4 v[P];
#pragma unroll
          for (int h = 0; h < P; ++h) v[h] = x_keep<T, AL>(cols[i & 1].v[q][h], kt * 128 + q * 32 + g * 8 + h * E, a.k);
          if constexpr (kF32) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __builtin_bit_cast(f32x4, v[e / 4])[e % 4];
            uint4 pl[3];
            split_planes(f, pl);
#pragma unroll
            for (int n = 0; n < 3; ++n) xf[q][n] = __builtin_bit_cast(u32x4, pl[n]);
          } else {
            xf[q][0] = v[0];
          }
        }
        multiply<T, GP, RT, 1>(tile[i], over,
                               [&](int q, u32x4(&f)[1][NX]) {
#pragma unroll
                                 for (int n = 0; n < NX; ++n) f[0][n] = xf[q][n];
                               },
                               acc);
        fetch(i, kt + D * NW);
      }
    }
  }
  constexpr int N = RT * 16;
#pragma unroll
  for (int t = 0; t < RT; ++t) *reinterpret_cast<f32x4*>(lds + (wave * 16 + j) * N + t * 16 + g * 4) = acc[t][0];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * N; i += NW * 64) {
    const int row = row0 + i / N, o = ot * 16 + i % N;
    if (row >= a.m || o >= a.o) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += lds[w * 16 * N + i];
    if (a.bias) s += to_f32(reinterpret_cast<const T*>(a.bias)[static_cast<int64_t>(model) * a.o + o]);
    reinterpret_cast<T*>(a.y)[(static_cast<int64_t>(model) * a.m + row) * a.o + o] = from_f32<T>(s);
  }
}

// More rows, through LDS: a workgroup of 8 or 16 waves, WR of them over output rows (RT tiles each) and WK over columns,
// brings CK tiles of 128 columns of x at a time, split into planes (fp32), once for all its output rows.  Weights come straight into registers, D tiles ahead of their use.
constexpr int kPad = 136;          // 16-bit values in a staged row: 128, and 8 that move the rows to other banks

template <typename T, int GP, int MT, int RT, int WR, int WK, int CK, bool AL>
__global__ __launch_bounds__(WR * WK * 64) void linear4_rows_kernel(Linear4 a) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int NX = kF32 ? 3 : 1, M = MT * 16, NT = WR * WK * 64;
  static_assert(CK % WK == 0, "every wave has whole tiles of a chunk");
  constexpr int PER = CK / WK, D = PER < 2 ? PER : 2;                   // tiles of a wave in a chunk; in flight
  constexpr int PC = CK * M * 16 / NT, E = 16 / sizeof(T), P = 8 / E;   // pieces of 8 columns of a row each thread brings
  static_assert(PER % D == 0 && CK * M * 16 % NT == 0, "slots repeat with the chunk, pieces with the threads");
  extern __shared__ float lds[];
  uint16_t* xs = reinterpret_cast<uint16_t*>(lds);                      // [CK][NX][M][kPad]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j = lane & 15, g = lane >> 4;
  const int wr = wave / WK, wk = wave % WK;
  const uint32_t model = fdiv(blockIdx.x, a.by_wg);
  const int ot0 = (blockIdx.x - model * a.by_wg.d) * (WR * RT) + wr * RT;
  const int row0 = a.m0 + blockIdx.y * M;
  const uint32_t over = bits_over<T>();

  // piece i of a thread: row r % M of tile r / M, r = tid / 16 + i NT / 16, columns 8 (tid % 16)
  u32x4 xr[PC][P];
  const T* src[PC];
#pragma unroll
  for (int i = 0; i < PC; ++i) src[i] = x_row<T>(a, model, row0 + (tid / 16 + i * (NT / 16)) % M);
  auto bring = [&](int kt0) {
#pragma unroll
    for (int i = 0; i < PC; ++i)
#pragma unroll
      for (int h = 0; h < P; ++h)
        xr[i][h] = x_load<T, AL>(src[i], (kt0 + (tid / 16 + i * (NT / 16)) / M) * 128 + (tid % 16) * 8 + h * E, a.k);
  };
  auto stage = [&](int kt0) {
#pragma unroll
    for (int i = 0; i < PC; ++i) {
      const int p = tid / 16 + i * (NT / 16), r = p % M, k = p / M, c = tid % 16;
      uint16_t* dst = xs + (k * NX * M + r) * kPad + c * 8;
      u32x4 v[P];
#pragma unroll
      for (int h = 0; h < P; ++h) v[h] = x_keep<T, AL>(xr[i][h], (kt0 + k) * 128 + c * 8 + h * E, a.k);
      if constexpr (kF32) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __builtin_bit_cast(f32x4, v[e / 4])[e % 4];
        uint4 pl[3];
        split_planes(f, pl);
#pragma unroll
        for (int n = 0; n < 3; ++n) *reinterpret_cast<uint4*>(dst + n * M * kPad) = pl[n];
      } else {
        *reinterpret_cast<u32x4*>(dst) = v[0];
      }
    }
  };

  f32x4 acc[RT][MT] = {};
  Tile<T, GP> tile[D][RT];
  auto fetch = [&](int slot, int kt) {
#pragma unroll
    for (int t = 0; t < RT; ++t) TileSource<T, GP>(a, model, ot0 + t, lane).load(tile[slot][t], kt);
  };
  bring(0);
#pragma unroll
  for (int i = 0; i < D; ++i) fetch(i, i * WK + wk);
  for (int kt0 = 0; kt0 < a.ktiles; kt0 += CK) {
    if (kt0) __syncthreads();
    stage(kt0);
    __syncthreads();
    if (kt0 + CK < a.ktiles) bring(kt0 + CK);
    // not unrolled further than the slots ask: code that runs once is fetched from memory as it runs
#pragma unroll 1
    for (int i0 = 0; i0 < PER; i0 += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int i = i0 + d, ct = i * WK + wk;            // tile of the chunk
        if (kt0 + ct < a.ktiles) {
          const uint16_t* x = xs + ct * NX * M * kPad + j * kPad + g * 8;
          multiply<T, GP, RT, MT>(tile[d], over,
                                  [&](int q, u32x4(&f)[MT][NX]) {
#pragma unroll
                                    for (int t = 0; t < MT; ++t)
#pragma unroll
                                      for (int n = 0; n < NX; ++n)
                                        f[t][n] = *reinterpret_cast<const u32x4*>(x + (n * M + t * 16) * kPad + q * 32);
                                  },
                                  acc);
        }
        fetch(d, i + D < PER ? kt0 + ct + D * WK : kt0 + CK + (i + D - PER) * WK + wk);
      }
    }
  }

  T* y = reinterpret_cast<T*>(a.y) + static_cast<int64_t>(model) * a.m * a.o;
  const T* bias = a.bias ? reinterpret_cast<const T*>(a.bias) + static_cast<int64_t>(model) * a.o : nullptr;
  __syncthreads();                   // x is done with: [WR][WK][M][RT * 16]
  constexpr int N = RT * 16;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t)
      *reinterpret_cast<f32x4*>(lds + (wave * M + t * 16 + j) * N + r * 16 + g * 4) = acc[r][t];
  __syncthreads();
  for (int i = tid; i < WR * M * N / 4; i += NT) {
    // neighbouring threads: neighbouring outputs of one row, four each
    const int c = i % (WR * N / 4) * 4, v = c / N, mr = i / (WR * N / 4);
    const int row = row0 + mr, o = (blockIdx.x - model * a.by_wg.d) * (WR * N) + c;
    if (row >= a.m || o >= a.o) continue;
    f32x4 s = {};
#pragma unroll
    for (int k = 0; k < WK; ++k) s += *reinterpret_cast<const f32x4*>(lds + ((v * WK + k) * M + mr) * N + c % N);
    store4(y + static_cast<int64_t>(row) * a.o, o, a.o, bias, s);
  }
}

// Calls go(m0, tiles of rows from m0) for grids of at most 65535 tiles of rows
template <typename F>
void over_rows(Linear4& a, int rows, F go) {
  for (int64_t m0 = 0; m0 < a.m; m0 += 65535ll * rows) {
    a.m0 = static_cast<int32_t>(m0);
    go(static_cast<uint32_t>(std::min<int64_t>(cdiv(a.m - m0, rows), 65535)));
  }
}

template <typename T, int GP, int RT, int NW>
void launch_few(Linear4 a, int64_t n, hipStream_t s) {
  const int64_t per = cdiv(a.otiles, RT);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(per));
  const auto kernel = a.vec ? linear4_few_kernel<T, GP, RT, NW, true> : linear4_few_kernel<T, GP, RT, NW, false>;
  over_rows(a, 16, [&](uint32_t tiles) { kernel<<<dim3(static_cast<uint32_t>(n * per), tiles), NW * 64, 0, s>>>(a); });
}

template <typename T, int GP, int MT, int RT, int WR, int WK, int CK>
void launch_rows(Linear4 a, int64_t n, hipStream_t s) {
  constexpr int NX = sizeof(T) == 4 ? 3 : 1, M = MT * 16;
  const int64_t per = cdiv(a.otiles, WR * RT);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(per));
  const size_t staged = CK * NX * M * kPad * 2, joined = WR * WK * M * RT * 16 * 4;
  const size_t lds = std::max(staged, joined);
  const auto kernel = a.vec ? linear4_rows_kernel<T, GP, MT, RT, WR, WK, CK, true> : linear4_rows_kernel<T, GP, MT, RT, WR, WK, CK, false>;
  if (lds > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
  over_rows(a, M, [&](uint32_t tiles) { kernel<<<dim3(static_cast<uint32_t>(n * per), tiles), WR * WK * 64, lds, s>>>(a); });
}

// Which kernel, for `tiles` tiles of output rows of all models and `rows` tiles of 16 rows of x (us on an MI355X,
// launches of a graph, weights from memory, bf16, groups of 128 where nothing else is said).
//
// Few tiles: a tile for each workgroup, its waves share the columns (64 tiles, 16 rows, K 2048: 6.6; through LDS 7.5; 8 waves
// where columns are long: 256 tiles, K 4096: 6.2, with 4 waves 6.5, with two tiles a workgroup 7.5), then two that share what
// they bring of x, for 8 waves where their workgroups all find room at once, which takes 128 registers (1024 tiles, K 4096:
// 12.6; for 4 waves 13.6; one tile for 4 waves 14.1; in fp16 with groups of 64: 12.6, 13.8, 14.2).  There is less room with
// groups of 32 (K 2048: 12.8 with 8, 10.9 with 4), and in bf16 with groups of 64 where x isn't whole vectors (K 2047: 14.4
// with 8, 13.0 with 4).
//
// More go through LDS.  16 waves fill a unit, with as much of x and W as registers take, where their workgroups come to
// whole rounds of all units, nearly; else 8 waves with 32 rows, of which a unit has two; else as many workgroups as can be:
//                                 16 waves, 64 rows   16 waves, 32 rows   8 waves, 32 rows   4 x 2 waves, 32 rows
//   4096 tiles, 64 rows, K 2048         42                  54                  51                 62
//   2048 tiles, 64 rows, K 2048         31                  26                  26                 33
//   1235 tiles, 64 rows, K 2048         29                  23                  23                 23
//   1235 tiles, 200 rows, K 2048        58                  63                  55                 63
//    512 tiles, 64 rows, K 2048         27                  21                  14                 11
// and by the same reasons in fp32, whose three planes of x leave less room.  Sixteen rows or fewer: 16 waves again where
// they come to whole rounds (4096 tiles, K 2048: 23, of 4 x 2 waves 27), and two waves over two tiles, without LDS,
// where there are too few columns for it to pay (1235 tiles, K 1024: 9.2 against 9.7; K 2048: 13.3 against 12.2).
template <typename T, int GP, int MT, int RT, int WR, int WK, int CK>
bool launch_if_full(const Linear4& a, int64_t n, hipStream_t s) {
  const int64_t wgs = n * cdiv(a.otiles, WR * RT) * cdiv(a.m, MT * 16);
  if (wgs * 5 < cdiv(wgs, 256) * 256 * 4) return false;              // the last round included, 4 of 5 units at work
  launch_rows<T, GP, MT, RT, WR, WK, CK>(a, n, s);
  return true;
}
template <typename T, int GP>
void dispatch(const Linear4& a, int64_t n, hipStream_t s) {
  constexpr bool F32 = sizeof(T) == 4;
  const int64_t tiles = n * a.otiles, rows = cdiv(a.m, 16);
  if (tiles * rows <= 256 && a.ktiles >= 32) return launch_few<T, GP, 1, 8>(a, n, s);
  if (tiles * rows <= 256) return launch_few<T, GP, 1, 4>(a, n, s);
  const bool room = !F32 && (GP == 1 || (GP == 2 && (a.vec || std::is_same<T, f16>::value)));
  if (rows == 1 && tiles <= (room ? 1024 : 512)) return launch_few<T, GP, 2, 8>(a, n, s);
  if (rows == 1 && tiles <= 1024) return launch_few<T, GP, 2, 4>(a, n, s);
  if constexpr (F32) {
    if (rows > 1 && launch_if_full<T, GP, 2, 2, 8, 1, 1>(a, n, s)) return;
    if (launch_if_full<T, GP, 1, 1, 16, 1, 4>(a, n, s)) return;
    if (tiles * rows > 1024) return launch_rows<T, GP, 1, 1, 8, 1, 2>(a, n, s);
    launch_rows<T, GP, 1, 1, 4, 2, 4>(a, n, s);
  } else {
    if (rows > 2 && launch_if_full<T, GP, 4, 1, 16, 1, 2>(a, n, s)) return;
    if (rows > 1 && launch_if_full<T, GP, 2, 1, 16, 1, 4>(a, n, s)) return;
    if (rows > 1 && (tiles * cdiv(rows, 2) > 1024 || a.ktiles <= 4)) return launch_rows<T, GP, 2, 1, 8, 1, 2>(a, n, s);
    if (rows > 2) return launch_rows<T, GP, 2, 1, 4, 2, 8>(a, n, s);
    if (rows == 1 && launch_if_full<T, GP, 1, 1, 16, 1, 8>(a, n, s)) return;
    if (rows == 1 && a.ktiles <= 8) return launch_few<T, GP, 2, 2>(a, n, s);
    launch_rows<T, GP, 1, 1, 4, 2, 16>(a, n, s);
  }
}

template <typename T>
void dispatch(const Linear4& a, int64_t n, int group, hipStream_t s) {
  if (group == 128)
    dispatch<T, 1>(a, n, s);
  else if (group == 64)
    dispatch<T, 2>(a, n, s);
  else
    dispatch<T, 4>(a, n, s);
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
  WC_REQUIRE(p.x && p.codes && p.scales && p.zeros && p.y, WC_ERR_NULL, "%s: null pointer", what);
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
  a.by_rows = make_fastdiv(static_cast<uint32_t>(p.x_rows_inner));
  // whole vectors: of 8 columns in 16 bits, of 4 in fp32
  a.vec = p.k * es % 16 == 0 && aligned(p.x, 16) && ubytes(p.x_stride_n, es) % 16 == 0 &&
                  ubytes(p.x_stride_outer, es) % 16 == 0 && ubytes(p.x_stride_inner, es) % 16 == 0;
  const hipStream_t s = as_stream(stream);
  if (p.dtype == WC_F32)
    dispatch<float>(a, p.n, p.group, s);
  else if (p.dtype == WC_BF16)
    dispatch<bf16>(a, p.n, p.group, s);
  else
    dispatch<f16>(a, p.n, p.group, s);
  return check_launch(what);
}
