// RMS norm of query and key heads with the rotation by position in the same pass.
//
//   y = x / sqrt(mean x^2 + eps) * w,   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)
//
// A pair of columns turns by 2 pi pos f, f turns per position, at most 1 / 2 pi.  pos f is taken in fp64, off by
// 2^-52 of itself with f's own rounding, and only its fraction of a turn goes on in fp32, its rounding's remainder after
// it (without: 2^-25 of a turn, more than fp32's cosines and sines are off by themselves), so that a token at any position
// up to 2^28 turns as exactly as the first (in fp32 the product itself would be off by 2^-24 of pos f turns).
//
// Memory bounds it: rows in, rows out, some 8 flops a value.  4 models' 4096 tokens of 32 + 8 heads of 128 columns in
// bf16, 335 MB: 70 us, 4.8 TB/s (a large copy here: 4.7 to 5.1).
//
// Both halves of a pair belong to one lane: it loads V columns from each half (V neighbouring pairs when
// pairs are neighbours), so a row needs no exchange but the sum of its squares.  A workgroup takes some
// tokens of one model: their cosines and sines are computed once, one thread a pair, and kept in LDS for all
// the heads.
#include <algorithm>

#include "wc_common.h"
#include "wc_serve_abi.h"

namespace wc {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;        // rows in flight per group of lanes (those 335 MB: 70 us; one row 72, four 80)

struct HeadNorm {
  const char *q, *k, *qw, *kw, *pos;
  char *qo, *ko;
  const double* freq;
  int64_t qs[4], ks[4], ps[3];
  int32_t hq, heads, dh, rot, tokens, tile, chunk, lanes_log2, pos8, pdt;
  FastDiv by_t, by_chunk, by_pairs;
  float eps, inv_dh;
};

__device__ __forceinline__ float param(const char* w, int64_t i, int dt) {
  if (dt == WC_F32) return reinterpret_cast<const float*>(w)[i];
  if (dt == WC_BF16) return to_f32(reinterpret_cast<const bf16*>(w)[i]);
  return to_f32(reinterpret_cast<const f16*>(w)[i]);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// The two column ranges of pairs [p, p + V): neighbours (interleaved), else one in each half of the turned
// columns, or of those that are not turned.
template <int V, bool INTER>
__device__ __forceinline__ void columns(const HeadNorm& a, int p, int& c0, int& c1) {
  if (INTER) {
    c0 = 2 * p;
    c1 = c0 + V;
    return;
  }
  const int half = a.rot >> 1;
  if (p < half) {
    c0 = p;
    c1 = p + half;
  } else {
    c0 = p + half;
    c1 = c0 + ((a.dh - a.rot) >> 1);
  }
}

// NC: groups of V pairs per lane
template <typename T, int V, int NC, bool INTER>
__global__ __launch_bounds__(kThreads) void head_norm_kernel(HeadNorm a) {
  extern __shared__ float lds[];
  const int pairs = a.dh >> 1;
  float2* turn = reinterpret_cast<float2*>(lds);            // [tile][pairs]: cos, sin
  float* weight = lds + 2 * a.tile * pairs;                 // [2][dh]
  const int tid = threadIdx.x;
  const int64_t model = blockIdx.z;
  const int tok0 = blockIdx.x * a.tile;
  const int toks = min(a.tile, a.tokens - tok0);
  const int head0 = blockIdx.y * a.chunk;
  const int heads = min(a.chunk, a.heads - head0);
  const int lanes = 1 << a.lanes_log2, lane = tid & (lanes - 1), group = tid >> a.lanes_log2;
  const int groups = kThreads >> a.lanes_log2;
  const int rows = toks * a.chunk;

  Vec<T, V> x[kUnroll][NC][2];
  auto load = [&](int r, Vec<T, V>(&v)[NC][2]) {
    const int tk = fdiv(r, a.by_chunk), hh = r - tk * a.chunk;
    if (r >= rows || hh >= heads) return false;
    const uint32_t tok = tok0 + tk, bb = fdiv(tok, a.by_t), tt = tok - bb * a.by_t.d;
    const int h = head0 + hh;
    const char* base = h < a.hq ? a.q + (model * a.qs[0] + bb * a.qs[1] + tt * a.qs[2] + h * a.qs[3]) * sizeof(T)
                                : a.k + (model * a.ks[0] + bb * a.ks[1] + tt * a.ks[2] + (h - a.hq) * a.ks[3]) * sizeof(T);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int p = (lane + c * lanes) * V;
      if (p < pairs) {
        int c0, c1;
        columns<V, INTER>(a, p, c0, c1);
        v[c][0] = *reinterpret_cast<const Vec<T, V>*>(base + c0 * sizeof(T));
        v[c][1] = *reinterpret_cast<const Vec<T, V>*>(base + c1 * sizeof(T));
      }
    }
    return true;
  };

  bool has[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) has[u] = load(group + u * groups, x[u]);

  for (int i = tid; i < 2 * a.dh; i += kThreads)
    weight[i] = i < a.dh ? param(a.qw, model * a.dh + i, a.pdt) : param(a.kw, model * a.dh + i - a.dh, a.pdt);
  for (int i = tid; i < toks * pairs; i += kThreads) {
    const int tk = fdiv(i, a.by_pairs), p = i - tk * pairs;
    float2 cs = make_float2(1.f, 0.f);
    if (p < (a.rot >> 1)) {
      const uint32_t tok = tok0 + tk, bb = fdiv(tok, a.by_t), tt = tok - bb * a.by_t.d;
      const int64_t at = model * a.ps[0] + bb * a.ps[1] + tt * a.ps[2];
      const int64_t pos = a.pos8 ? reinterpret_cast<const int64_t*>(a.pos)[at] : reinterpret_cast<const int32_t*>(a.pos)[at];
      double turns = static_cast<double>(pos) * a.freq[p];
      turns -= rint(turns);
      const float half_turns = static_cast<float>(2.0 * turns);
      float sn, cn;
      sincospif(half_turns, &sn, &cn);
      // what that rounding left of the angle, under 2^-23: sine and cosine of it are itself and 1
      const float rest = static_cast<float>(2.0 * turns - half_turns) * 3.14159265f;
      cs = make_float2(fmaf(-rest, sn, cn), fmaf(rest, cn, sn));
    }
    turn[i] = cs;
  }
  __syncthreads();

  // columns that aren't turned are left alone by their neighbours, whatever those hold
  const bool some_rest = a.rot < a.dh;
  for (int r0 = group; r0 < rows; r0 += kUnroll * groups) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = r0 + u * groups;
      float v[NC][2][V], ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const bool on = (lane + c * lanes) * V < pairs;
          v[c][0][e] = on ? to_f32(x[u][c][0].v[e]) : 0.f;
          v[c][1][e] = on ? to_f32(x[u][c][1].v[e]) : 0.f;
          ss += v[c][0][e] * v[c][0][e] + v[c][1][e] * v[c][1][e];
        }
      for (int off = lanes >> 1; off; off >>= 1) ss += __shfl_xor(ss, off, 64);
      if (!has[u]) continue;
      const float inv = 1.f / sqrtf(ss * a.inv_dh + a.eps);
      const int tk = fdiv(r, a.by_chunk), h = head0 + r - tk * a.chunk;
      const int64_t tok = model * a.tokens + tok0 + tk;
      char* out = h < a.hq ? a.qo + (tok * a.hq + h) * a.dh * sizeof(T)
                           : a.ko + (tok * (a.heads - a.hq) + h - a.hq) * a.dh * sizeof(T);
      const float* w = weight + (h < a.hq ? 0 : a.dh);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int p = (lane + c * lanes) * V;
        if (p >= pairs) continue;
        int c0, c1;
        columns<V, INTER>(a, p, c0, c1);
        float y[2][V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          y[0][e] = v[c][0][e] * inv * w[c0 + e];
          y[1][e] = v[c][1][e] * inv * w[c1 + e];
        }
        Vec<T, V> o0, o1;
        const float2* cs = turn + tk * pairs + p;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          // interleaved: pair e is values 2e and 2e + 1 of the 2V
          const float s = INTER ? y[(2 * e) / V][(2 * e) % V] : y[0][e];
          const float t = INTER ? y[(2 * e + 1) / V][(2 * e + 1) % V] : y[1][e];
          float s2 = s * cs[e].x - t * cs[e].y, t2 = t * cs[e].x + s * cs[e].y;
          if (some_rest && p + e >= (a.rot >> 1)) s2 = s, t2 = t;
          if (INTER) {
            ((2 * e) / V ? o1 : o0).v[(2 * e) % V] = from_f32<T>(s2);
            ((2 * e + 1) / V ? o1 : o0).v[(2 * e + 1) % V] = from_f32<T>(t2);
          } else {
            o0.v[e] = from_f32<T>(s2);
            o1.v[e] = from_f32<T>(t2);
          }
        }
        *reinterpret_cast<Vec<T, V>*>(out + c0 * sizeof(T)) = o0;
        *reinterpret_cast<Vec<T, V>*>(out + c1 * sizeof(T)) = o1;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) has[u] = load(r0 + (kUnroll + u) * groups, x[u]);
  }
}

template <typename T, int V, int NC>
void launch(const HeadNorm& a, bool inter, dim3 grid, size_t lds, hipStream_t s) {
  if (inter)
    head_norm_kernel<T, V, NC, true><<<grid, kThreads, lds, s>>>(a);
  else
    head_norm_kernel<T, V, NC, false><<<grid, kThreads, lds, s>>>(a);
}

template <typename T>
void dispatch(const HeadNorm& a, int v, bool inter, dim3 grid, size_t lds, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (v == 8) return launch<T, 8, 1>(a, inter, grid, lds, s);
  if (v == 4) return launch<T, 4, 1>(a, inter, grid, lds, s);
  if (v == 2) return launch<T, 2, 1>(a, inter, grid, lds, s);
  launch<T, 1, 2>(a, inter, grid, lds, s);
}

}  // namespace
}  // namespace wc

extern "C" int32_t wc_serve_abi_version(void) { return WC_SERVE_ABI_VERSION; }

extern "C" int32_t wc_head_norm_rotary(const wc_head_norm_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_head_norm_rotary";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_head_norm_args& p = *args;
  const int es = dtype_size(p.dtype);
  WC_REQUIRE(es && dtype_size(p.param_dtype), WC_ERR_DTYPE, "%s: dtype %d / %d", what, p.dtype, p.param_dtype);
  WC_REQUIRE(p.position_bytes == 4 || p.position_bytes == 8, WC_ERR_DTYPE, "%s: positions of %d bytes", what,
             p.position_bytes);
  WC_REQUIRE(p.n >= 0 && p.b >= 0 && p.t >= 0 && p.q_heads >= 0 && p.k_heads >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(p.head_dim > 0 && p.head_dim % 2 == 0 && p.rotary_dim >= 0 && p.rotary_dim % 2 == 0 && p.rotary_dim <= p.head_dim,
             WC_ERR_SHAPE, "%s: head_dim %lld and rotary_dim %lld must be even, rotary_dim at most head_dim", what,
             (long long)p.head_dim, (long long)p.rotary_dim);
  WC_REQUIRE(p.head_dim <= 256, WC_ERR_LIMIT, "%s: head_dim %lld above 256", what, (long long)p.head_dim);
  const int64_t tokens = mul_sat({p.b, p.t});
  WC_REQUIRE(p.n <= 65535 && p.q_heads <= 32767 && p.k_heads <= 32767 && tokens < (1ll << 24), WC_ERR_LIMIT,
             "%s: more than 65535 models, 32767 heads or 2^24 tokens per model", what);
  const int64_t heads = p.q_heads + p.k_heads;
  WC_REQUIRE(mul_sat({p.n, tokens, heads, p.head_dim, 8}) < INT64_MAX, WC_ERR_LIMIT, "%s: sizes overflow", what);
  if (p.n == 0 || tokens == 0 || heads == 0) return WC_OK;
  WC_REQUIRE((p.q_heads == 0 || (p.q && p.q_out && p.q_weight)) && (p.k_heads == 0 || (p.k && p.k_out && p.k_weight)) &&
                 (p.rotary_dim == 0 || (p.freq && p.positions)),
             WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(aligned(p.q, es) && aligned(p.k, es) && aligned(p.q_out, es) && aligned(p.k_out, es) && aligned(p.freq, 8) &&
                 aligned(p.positions, p.position_bytes),
             WC_ERR_ALIGN, "%s: pointers must be aligned to their elements", what);
  // the widest vector that every row and both halves of the pairs are whole multiples of
  int v = 16 / es;
  auto fits = [&](int w) {
    const uint64_t vb = static_cast<uint64_t>(w) * es;
    if (p.interleaved ? (p.head_dim / 2) % w != 0 : (p.rotary_dim / 2) % w != 0 || ((p.head_dim - p.rotary_dim) / 2) % w != 0)
      return false;
    for (const void* ptr : {p.q, p.k, static_cast<const void*>(p.q_out), static_cast<const void*>(p.k_out)})
      if (!aligned(ptr, static_cast<int64_t>(vb))) return false;
    for (int64_t s : {p.q_stride_n, p.q_stride_b, p.q_stride_t, p.q_stride_h, p.k_stride_n, p.k_stride_b, p.k_stride_t, p.k_stride_h})
      if (ubytes(s, es) % vb != 0) return false;
    return true;
  };
  while (v > 1 && !fits(v)) v >>= 1;

  HeadNorm a;
  a.q = static_cast<const char*>(p.q);
  a.k = static_cast<const char*>(p.k);
  a.qo = static_cast<char*>(p.q_out);
  a.ko = static_cast<char*>(p.k_out);
  a.qw = static_cast<const char*>(p.q_heads ? p.q_weight : p.k_weight);
  a.kw = static_cast<const char*>(p.k_heads ? p.k_weight : p.q_weight);
  a.pos = static_cast<const char*>(p.positions);
  a.freq = p.freq;
  const int64_t qs[4] = {p.q_stride_n, p.q_stride_b, p.q_stride_t, p.q_stride_h};
  const int64_t ks[4] = {p.k_stride_n, p.k_stride_b, p.k_stride_t, p.k_stride_h};
  const int64_t ps[3] = {p.p_stride_n, p.p_stride_b, p.p_stride_t};
  for (int i = 0; i < 4; ++i) a.qs[i] = qs[i], a.ks[i] = ks[i];
  for (int i = 0; i < 3; ++i) a.ps[i] = ps[i];
  a.hq = static_cast<int32_t>(p.q_heads);
  a.heads = static_cast<int32_t>(heads);
  a.dh = static_cast<int32_t>(p.head_dim);
  a.rot = static_cast<int32_t>(p.rotary_dim);
  a.tokens = static_cast<int32_t>(tokens);
  a.pos8 = p.position_bytes == 8;
  a.pdt = p.param_dtype;
  a.eps = p.eps;
  a.inv_dh = 1.f / static_cast<float>(a.dh);
  const int pairs = a.dh / 2, need = static_cast<int>(cdiv(pairs, v));
  a.lanes_log2 = 0;
  while ((1 << a.lanes_log2) < need && a.lanes_log2 < 6) ++a.lanes_log2;
  // A workgroup takes about 4 rows per group of lanes, all heads of some tokens or a part of the heads, or fewer where
  // that would leave compute units without work (us on an MI355X, 8 heads of 128 columns for 32 heads of queries, bf16:
  // 4 models of 4096 tokens 70 with 4 rows, 76 with 2, 77 with 8; 8 models of 4 tokens 7.1 with 4, 5.0 with 2)
  int target = 4 * (kThreads >> a.lanes_log2);
  for (;; target >>= 1) {
    a.chunk = std::min(a.heads, target);
    a.tile = std::min({std::max(1, target / a.chunk), 4096 / pairs, a.tokens});    // at most 32 KB of cosines and sines
    if (target <= kThreads >> a.lanes_log2 || p.n * cdiv(a.tokens, a.tile) * cdiv(a.heads, a.chunk) >= 256) break;
  }
  a.by_t = make_fastdiv(static_cast<uint32_t>(p.t));
  a.by_chunk = make_fastdiv(static_cast<uint32_t>(a.chunk));
  a.by_pairs = make_fastdiv(static_cast<uint32_t>(pairs));
  const dim3 grid(static_cast<uint32_t>(cdiv(a.tokens, a.tile)), static_cast<uint32_t>(cdiv(a.heads, a.chunk)),
                  static_cast<uint32_t>(p.n));
  const size_t lds = static_cast<size_t>(2 * a.tile * pairs + 2 * a.dh) * sizeof(float);
  const hipStream_t s = as_stream(stream);
  const bool inter = p.interleaved != 0;
  if (p.dtype == WC_F32)
    dispatch<float>(a, v, inter, grid, lds, s);
  else if (p.dtype == WC_BF16)
    dispatch<bf16>(a, v, inter, grid, lds, s);
  else
    dispatch<f16>(a, v, inter, grid, lds, s);
  return check_launch(what);
}
