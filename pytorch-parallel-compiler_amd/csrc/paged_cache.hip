// Writing rows into a paged key-value cache, as they are or as 8-bit codes, and reading them back.
//
// One group of lanes has a row: head_dim values of one head of one token, 16 bytes of them a lane.  Both
// kernels only move rows, so they are bound by memory; what decides is that every access is a whole vector
// and that enough of them are in flight.  16 sequences' 750 to 1500 new tokens of 8 heads of 128 columns in bf16:
// written as they are (154 MB) 26 us, 6.0 TB/s; as codes (112 MB) 32 us, which the search for each row's scale and the
// codes' arithmetic keep from 25; codes read back (145 MB) 26 us, 5.5 TB/s.
//
// 8 bits: scale = max(max |x| / 127, 2^-126) (one unit less for fp32's largest value), code = x / scale to the nearest, ties to even.  The quotient is
// never formed: c = x * (1 / scale) to the nearest is off by at most one, and then only next to a half; the remainder
// x - c scale is exact (one fused multiply-add whose result fits 24 bits) and its place against scale / 2
// puts c right, for the lanes that have such a value.  The code is so a function of x and scale alone.
#include <algorithm>

#include "wc_paged.h"

namespace wc {
namespace {

constexpr int kThreads = 256;
constexpr float kMost = 0x1.020406p121f;      // the largest scale: 127 of the next one round to infinity in fp32
constexpr int kRows = 4;           // rows of a group of lanes, all on their way at once (those codes written and read: 61 us;
                                   // one row 68, two 64, eight 73)

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

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

// The largest magnitude of a lane's values as the bits of a float, under which an infinity or NaN is larger than any
// finite value; 16-bit values are compared two at a time.
template <typename T, int V, int NC>
__device__ __forceinline__ uint32_t largest(const Vec<T, V> (&x)[NC]) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  uint32_t top = 0;
  if constexpr (sizeof(T) == 2 && V == 8) {
    u16x2 t = {};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const u32x4 w = __builtin_bit_cast(u32x4, x[c]);
#pragma unroll
      for (int e = 0; e < 4; ++e) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, static_cast<uint32_t>(w[e]) & 0x7fff7fffu));
    }
    const uint16_t m = max(t[0], t[1]);
    top = __builtin_bit_cast(uint32_t, to_f32(__builtin_bit_cast(T, m)));
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) top = max(top, __builtin_bit_cast(uint32_t, to_f32(x[c].v[e])) & 0x7fffffffu);
  }
  return top;
}

struct Write {
  PagedTable t;
  const char *src[2];
  char* pages[2];
  float* scales[2];
  int64_t stride[2][4];
  const int32_t *start, *count;
  int32_t steps, dh, row, lanes_log2;
  FastDiv by_b, by_tiles, by_heads;      // sequences per model; workgroups per sequence
};

// V: values a lane loads at once; NC: of those per lane
template <typename T, bool Q8, int V, int NC>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(Write a) {
  const int tid = threadIdx.x, kv = blockIdx.y;
  const int lanes = 1 << a.lanes_log2, lane = tid & (lanes - 1), groups = kThreads >> a.lanes_log2;
  const uint32_t seq = fdiv(blockIdx.x, a.by_tiles), tile = blockIdx.x - seq * a.by_tiles.d;
  const uint32_t model = fdiv(seq, a.by_b), b = seq - model * a.by_b.d;
  const int64_t* st = a.stride[kv];
  const T* src = reinterpret_cast<const T*>(a.src[kv]) + model * st[0] + b * st[1];
  const int start = a.start[seq];
  int n = a.steps;
  if (a.count) n = a.count[seq];
  if (start < 0) return;                 // whatever its count says
  if (n > a.steps) {
    n = a.steps;
    paged_fault(a.t);
  }
  const uint32_t rows = static_cast<uint32_t>(max(n, 0)) * a.t.heads;       // to write
  const uint32_t r0 = tile * (groups * kRows) + (tid >> a.lanes_log2);
  if (tile * (groups * kRows) >= rows) return;

  // rows past the last are loaded as the last and not stored; lanes past a row's end hold its first values again
  typedef typename std::conditional<V == 1, T, u32x4>::type Piece;      // an array of structs would not stay in registers
  Piece x[kRows][NC];
  int32_t row[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t r = min(r0 + u * groups, rows - 1), step = fdiv(r, a.by_heads), h = r - step * a.by_heads.d;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = (lane + c * lanes) * V;
      x[u][c] = *reinterpret_cast<const Piece*>(src + step * st[2] + h * st[3] + (d < a.dh ? d : 0));
    }
    row[u] = paged_entry(a.t, seq, start + step);                 // at most 2^32 - 2
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t r = min(r0 + u * groups, rows - 1), step = fdiv(r, a.by_heads), tok = start + step;
    row[u] = tok > INT32_MAX ? -1 : paged_row(a.t, row[u], tok, r - step * a.by_heads.d);
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const bool mine = r0 + u * groups < rows;
    if (mine && row[u] < 0) paged_fault(a.t);
    const bool store = mine && row[u] >= 0;
    const int64_t at = static_cast<int64_t>(row[u]) * a.row;
    if constexpr (!Q8) {
      if (!store) continue;
      T* dst = reinterpret_cast<T*>(a.pages[kv]) + at;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = (lane + c * lanes) * V;
        if (d < a.dh) *reinterpret_cast<Piece*>(dst + d) = x[u][c];
      }
      for (int d = a.dh + lane; d < a.row; d += lanes) dst[d] = static_cast<T>(0.f);
    } else {
      Vec<T, V> v[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) v[c] = __builtin_bit_cast(Vec<T, V>, x[u][c]);
      uint32_t top = largest<T, V, NC>(v);
      for (int off = lanes >> 1; off; off >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 64)));
      const bool finite = top < 0x7f800000u;
      const float scale = finite ? fminf(fmaxf(__builtin_bit_cast(float, top) / 127.f, 0x1p-126f), kMost) : __builtin_nanf("");
      const float inv = __builtin_amdgcn_rcpf(scale);
      uint32_t code[NC][V];
      float far = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float off;
          code[c][e] = code8(to_f32(v[c].v[e]), scale, inv, off);
          far = fmaxf(far, off);
        }
      // 2^-15 covers the product's rounding and inv's: 2^-22 of a quotient of up to 127
      if (far > scale * (0.5f - 0x1p-15f))
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) code[c][e] = code8_near_half(to_f32(v[c].v[e]), scale, inv);
      if (!store) continue;
      int8_t* dst = reinterpret_cast<int8_t*>(a.pages[kv]) + at;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = (lane + c * lanes) * V;
        if (d >= a.dh) continue;
        if constexpr (V == 1) {
          dst[d] = static_cast<int8_t>(finite ? code[c][0] : 0u);
        } else {
          Vec<uint32_t, V / 4> o;
#pragma unroll
          for (int q = 0; q < V / 4; ++q) {
            const uint32_t* k = code[c] + 4 * q;
            const uint32_t lo = __builtin_amdgcn_perm(k[1], k[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(k[3], k[2], 0x0c0c0400u);
            o.v[q] = finite ? lo | hi << 16 : 0u;
          }
          *reinterpret_cast<Vec<uint32_t, V / 4>*>(dst + d) = o;
        }
      }
      for (int d = a.dh + lane; d < a.row; d += lanes) dst[d] = 0;
      if (lane == 0) a.scales[kv][row[u]] = scale;
    }
  }
}

struct Read {
  PagedTable t;
  const char* pages[2];
  const float* scales[2];
  char* out[2];
  const int32_t* lengths;
  int32_t most, dh, row, lanes_log2;
  FastDiv by_tiles, by_heads;
};

template <typename T, bool Q8, int V, int NC>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(Read a) {
  typedef typename std::conditional<Q8, int8_t, T>::type S;
  const int tid = threadIdx.x, kv = blockIdx.y;
  const int lanes = 1 << a.lanes_log2, lane = tid & (lanes - 1), groups = kThreads >> a.lanes_log2;
  const uint32_t seq = fdiv(blockIdx.x, a.by_tiles), tile = blockIdx.x - seq * a.by_tiles.d;
  const uint32_t rows = static_cast<uint32_t>(a.most) * a.t.heads;
  const uint32_t r0 = tile * (groups * kRows) + (tid >> a.lanes_log2);
  const int32_t length = a.lengths[seq];
  if (length > a.most) paged_fault(a.t);
  int32_t row[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) row[u] = paged_entry(a.t, seq, fdiv(min(r0 + u * groups, rows - 1), a.by_heads));
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t r = min(r0 + u * groups, rows - 1), tok = fdiv(r, a.by_heads), h = r - tok * a.by_heads.d;
    const bool has = static_cast<int32_t>(tok) < length;
    row[u] = has ? paged_row(a.t, row[u], tok, h) : -1;
    if (has && row[u] < 0) paged_fault(a.t);
  }
  // rows that aren't there are read as row 0 of the pool, if it has one, and become zeros
  Vec<S, V> x[kRows][NC];
  float scale[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int64_t at = max(row[u], 0);
    if (a.t.pages == 0) continue;
    scale[u] = Q8 ? a.scales[kv][at] : 1.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = (lane + c * lanes) * V;
      x[u][c] = *reinterpret_cast<const Vec<S, V>*>(reinterpret_cast<const S*>(a.pages[kv]) + at * a.row + (d < a.dh ? d : 0));
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t r = r0 + u * groups;
    if (r >= rows) continue;
    T* out = reinterpret_cast<T*>(a.out[kv]) + (static_cast<int64_t>(seq) * rows + r) * a.dh;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = (lane + c * lanes) * V;
      if (d >= a.dh) continue;
      Vec<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (Q8)
          o.v[e] = from_f32<T>(row[u] < 0 ? 0.f : static_cast<float>(x[u][c].v[e]) * scale[u]);
        else
          o.v[e] = row[u] < 0 ? static_cast<T>(0.f) : x[u][c].v[e];
      }
      *reinterpret_cast<Vec<T, V>*>(out + d) = o;
    }
  }
}

int log2_lanes(int64_t need) {
  int l = 0;
  while ((1 << l) < need && l < 6) ++l;
  return l;
}

// Runs F<T, Q8, V, NC>: whole 16-byte vectors of T (a row of at most 256 values fits 64 lanes), else single values
template <template <typename, bool, int, int> class F, typename A>
void dispatch(int dtype, int bits, bool vec, const A& a, dim3 grid, hipStream_t s) {
  auto go = [&](auto t) {
    typedef decltype(t) T;
    constexpr int V = 16 / sizeof(T);
    if (bits == 8)
      vec ? F<T, true, V, 1>::run(a, grid, s) : F<T, true, 1, 4>::run(a, grid, s);
    else
      vec ? F<T, false, V, 1>::run(a, grid, s) : F<T, false, 1, 4>::run(a, grid, s);
  };
  if (dtype == WC_F32)
    go(float());
  else if (dtype == WC_BF16)
    go(bf16());
  else
    go(f16());
}
template <typename T, bool Q8, int V, int NC>
struct RunWrite {
  static void run(const Write& a, dim3 grid, hipStream_t s) { cache_write_kernel<T, Q8, V, NC><<<grid, kThreads, 0, s>>>(a); }
};
template <typename T, bool Q8, int V, int NC>
struct RunRead {
  static void run(const Read& a, dim3 grid, hipStream_t s) { cache_read_kernel<T, Q8, V, NC><<<grid, kThreads, 0, s>>>(a); }
};

}  // namespace
}  // namespace wc

extern "C" int32_t wc_cache_write(const wc_cache_write_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_cache_write";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_cache_write_args& p = *args;
  const wc_paged_cache& c = p.cache;
  if (int32_t rc = paged_check(c, what)) return rc;
  const int es = dtype_size(c.dtype);
  WC_REQUIRE(p.t >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(mul_sat({p.t, c.heads}) < (1ll << 30), WC_ERR_LIMIT, "%s: 2^30 rows per sequence or more", what);
  const int64_t seqs = c.n * c.b;
  if (seqs == 0 || p.t == 0 || c.heads == 0) return WC_OK;
  if (int32_t rc = paged_check_pointers(c, what)) return rc;
  WC_REQUIRE(p.k && p.v && p.start, WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(aligned(p.k, es) && aligned(p.v, es) && aligned(p.start, 4) && aligned(p.count, 4), WC_ERR_ALIGN,
             "%s: pointers must be aligned to their elements", what);
  Write a;
  a.t = paged_table(c, p.start);
  a.src[0] = static_cast<const char*>(p.k);
  a.src[1] = static_cast<const char*>(p.v);
  a.pages[0] = static_cast<char*>(c.k_pages);
  a.pages[1] = static_cast<char*>(c.v_pages);
  a.scales[0] = c.k_scales;
  a.scales[1] = c.v_scales;
  const int64_t st[2][4] = {{p.k_stride_n, p.k_stride_b, p.k_stride_t, p.k_stride_h},
                            {p.v_stride_n, p.v_stride_b, p.v_stride_t, p.v_stride_h}};
  bool vec = c.head_dim * es % 16 == 0 && aligned(p.k, 16) && aligned(p.v, 16);
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 4; ++j) {
      a.stride[i][j] = st[i][j];
      vec = vec && ubytes(st[i][j], es) % 16 == 0;
    }
  a.start = p.start;
  a.count = p.count;
  a.steps = static_cast<int32_t>(p.t);
  a.dh = static_cast<int32_t>(c.head_dim);
  a.row = static_cast<int32_t>(c.row);
  a.lanes_log2 = log2_lanes(vec ? cdiv(c.head_dim * es, 16) : c.head_dim);
  const int64_t tiles = cdiv(p.t * c.heads, kRows * (kThreads >> a.lanes_log2));
  WC_REQUIRE(mul_sat({tiles, seqs}) < (1ll << 32) / kThreads, WC_ERR_LIMIT, "%s: too many rows for one launch", what);
  a.by_b = make_fastdiv(static_cast<uint32_t>(c.b));
  a.by_tiles = make_fastdiv(static_cast<uint32_t>(tiles));
  a.by_heads = make_fastdiv(static_cast<uint32_t>(c.heads));
  dispatch<RunWrite>(c.dtype, c.bits, vec, a, dim3(static_cast<uint32_t>(tiles * seqs), 2), as_stream(stream));
  return check_launch(what);
}

extern "C" int32_t wc_cache_read(const wc_cache_read_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_cache_read";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_cache_read_args& p = *args;
  const wc_paged_cache& c = p.cache;
  if (int32_t rc = paged_check(c, what)) return rc;
  const int es = dtype_size(c.dtype);
  WC_REQUIRE(p.max_length >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(mul_sat({p.max_length, c.heads}) < (1ll << 30), WC_ERR_LIMIT, "%s: 2^30 rows per sequence or more", what);
  const int64_t seqs = c.n * c.b;
  if (seqs == 0 || p.max_length == 0 || c.heads == 0) return WC_OK;
  if (int32_t rc = paged_check_pointers(c, what)) return rc;
  WC_REQUIRE(p.k && p.v && p.lengths, WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(aligned(p.k, es) && aligned(p.v, es) && aligned(p.lengths, 4), WC_ERR_ALIGN,
             "%s: pointers must be aligned to their elements", what);
  Read a;
  a.t = paged_table(c, p.lengths);
  a.pages[0] = static_cast<const char*>(c.k_pages);
  a.pages[1] = static_cast<const char*>(c.v_pages);
  a.scales[0] = c.k_scales;
  a.scales[1] = c.v_scales;
  a.out[0] = static_cast<char*>(p.k);
  a.out[1] = static_cast<char*>(p.v);
  a.lengths = p.lengths;
  a.most = static_cast<int32_t>(p.max_length);
  a.dh = static_cast<int32_t>(c.head_dim);
  a.row = static_cast<int32_t>(c.row);
  const bool vec = c.head_dim * es % 16 == 0 && aligned(p.k, 16) && aligned(p.v, 16);
  a.lanes_log2 = log2_lanes(vec ? cdiv(c.head_dim * es, 16) : c.head_dim);
  const int64_t tiles = cdiv(p.max_length * c.heads, kRows * (kThreads >> a.lanes_log2));
  WC_REQUIRE(mul_sat({tiles, seqs}) < (1ll << 32) / kThreads, WC_ERR_LIMIT, "%s: too many rows for one launch", what);
  a.by_tiles = make_fastdiv(static_cast<uint32_t>(tiles));
  a.by_heads = make_fastdiv(static_cast<uint32_t>(c.heads));
  dispatch<RunRead>(c.dtype, c.bits, vec, a, dim3(static_cast<uint32_t>(tiles * seqs), 2), as_stream(stream));
  return check_launch(what);
}
