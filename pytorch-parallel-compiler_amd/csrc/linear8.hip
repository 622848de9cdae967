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

// 16 values of a row from column k on, zeros from its end on
template <typename T>
__device__ __forceinline__ void load16(const T* x, int k, int end, T (&v)[16]) {
  if (k + 16 <= end) {
    __builtin_memcpy(v, x + k, sizeof v);            // at element alignment
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = k + e < end ? x[k + e] : from_f32<T>(0.f);
  }
}

// Codes and scales of 16 rows of x: lane l has row l % 16 and columns 16 (l / 16).. of every tile of its wave, which is what
// it writes.  KEPT tiles a wave stay in registers between the search for the scale and the codes; rows longer than that
// are read a second time.
template <typename T, int NW, int KEPT>
__global__ __launch_bounds__(NW * 64) void linear8_codes_kernel(Linear8 a) {
  __shared__ uint32_t tops[NW][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const uint32_t model = fdiv(blockIdx.x, a.by_mtiles);
  const int mt = blockIdx.x - model * a.by_mtiles.d;
  const uint32_t r = min(mt * 16 + j, a.m - 1), outer = fdiv(r, a.by_rows);        // past the last: the last again
  const T* x = reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (r - outer * a.by_rows.d) * a.xi;
  T v[KEPT][16];
  auto top16 = [](const T(&t)[16], uint32_t top) {
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, __builtin_bit_cast(uint32_t, to_f32(t[e])) & 0x7fffffffu);
    return top;
  };
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < KEPT; ++i) load16(x, ((wave + i * NW) * 4 + g) * 16, a.k, v[i]);
#pragma unroll
  for (int i = 0; i < KEPT; ++i) top = top16(v[i], top);
  for (int t = wave + KEPT * NW; t < a.ktiles; t += NW) {
    T u[16];
    load16(x, (t * 4 + g) * 16, a.k, u);
    top = top16(u, top);
  }
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
  if (g == 0) tops[wave][j] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) top = max(top, tops[w][j]);
  const bool finite = top < 0x7f800000u;
  const float scale = finite ? row_scale(top) : __builtin_nanf("");
  const float inv = __builtin_amdgcn_rcpf(scale);
  if (threadIdx.x < 16) a.s[static_cast<int64_t>(blockIdx.x) * 16 + j] = scale;
  uint8_t* out = a.c + (static_cast<int64_t>(blockIdx.x) * a.ktiles) * 1024 + lane * 16;
  auto put = [&](const T(&t)[16], int tile) {
    uint32_t code[16];
    float far = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float off;
      code[e] = code8(to_f32(t[e]), scale, inv, off);
      far = fmaxf(far, off);
    }
    if (far > scale * kNearHalf)
#pragma unroll
      for (int e = 0; e < 16; ++e) code[e] = code8_near_half(to_f32(t[e]), scale, inv);
    u32x4 o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t* c = code + 4 * q;
      const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
      o[q] = finite ? lo | hi << 16 : 0u;
    }
    *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(tile) * 1024) = o;
  };
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
    if (wave + i * NW < a.ktiles) put(v[i], wave + i * NW);
  for (int t = wave + KEPT * NW; t < a.ktiles; t += NW) {
    T u[16];
    load16(x, (t * 4 + g) * 16, a.k, u);
    put(u, t);
  }
}

// outputs o..o + 3 of row r, those there are
template <typename T>
__device__ __forceinline__ void finish4(const Linear8& a, uint32_t model, int r, int o, i32x4 sum) {
  if (r >= a.m || o >= a.o) return;
  const int64_t at = static_cast<int64_t>(model) * a.o + o;
  const float s = a.s[static_cast<int64_t>(model) * a.mtiles * 16 + r];
  T* y = reinterpret_cast<T*>(a.y) + (static_cast<int64_t>(model) * a.m + r) * a.o + o;
  const T* bias = reinterpret_cast<const T*>(a.bias) + at;
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool in = o + e < a.o;
    const float f = static_cast<float>(sum[e]) * (s * a.scales[in ? at + e : at]);
    v[e] = from_f32<T>(a.bias ? f + to_f32(bias[in ? e : 0]) : f);
  }
  if (a.vec) {
    __builtin_memcpy(__builtin_assume_aligned(y, 4 * sizeof(T)), v, sizeof v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (o + e < a.o) y[e] = v[e];
  }
}

// Up to 16 rows of x: a workgroup has RT tiles of output rows, its waves every NW-th tile of columns, D of them on their way.
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
    finish4<T>(a, model, mt * 16 + (lane & 15), (ot0 + t) * 16 + (lane >> 4) * 4, sum);
  }
}

// Tiles of BM x BN outputs through LDS: WM x WN waves of FM x FN tiles each, NS stages of 128 columns in a ring, brought by DMA.
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
    __syncthreads();
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
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
      finish4<T>(a, model, (mt0 + wm + j) * 16 + (lane & 15), (ot0 + wn + i) * 16 + (lane >> 4) * 4, acc[i][j]);
}

template <typename T, int RT, int NW, int D>
void launch_few(Linear8 a, int64_t n, hipStream_t s) {
  const int64_t per = cdiv(a.otiles, RT);
  a.by_wg = make_fastdiv(static_cast<uint32_t>(per));
  linear8_few_kernel<T, RT, NW, D><<<dim3(static_cast<uint32_t>(n * per), static_cast<uint32_t>(a.mtiles)), NW * 64, 0, s>>>(a);
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
void launch(const Linear8& a, int64_t n, hipStream_t s) {
  const uint32_t tiles = static_cast<uint32_t>(n * a.mtiles);
  linear8_codes_kernel<T, 16, 4><<<tiles, 1024, 0, s>>>(a);
  if (a.mtiles == 1) return launch_few<T, 1, 4, 8>(a, n, s);
  if (a.mtiles <= 4) return launch_tile<T, 4, 2, 1, 4, 3>(a, n, s);
  launch_tile<T, 4, 4, 2, 2, 2>(a, n, s);
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
