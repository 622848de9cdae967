// Attention of one new token of every sequence over its pages of cached keys and values.
//
//   o = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),   s_i = scale q . k_i,   m the running maximum
//
// in one pass over the sequence.  A query head group shares a key head, so up to 16 query heads are the columns of
// one MFMA tile and every K and V row is read once for all of them.  What bounds it is that reading: 4 flops per
// stored value and query head, far under the machine's balance; the matrix instructions run mostly empty for
// small groups and still cost a tenth of the time their rows take to arrive.
//
// A wave takes 32 tokens at a time, and nothing but the sum over its lanes ever leaves its registers:
//   scores   S [token][query] = K Q^T, K rows as the A operand: lane l brings 16-byte pieces of token l % 16, Q the
//            same columns, so the order of columns inside the product is free and pieces are whole vectors.
//   softmax  the accumulator has query l % 16 and tokens 4 (l / 16) + r, of two tiles of 16 tokens.
//   output   O^T [column][query] = V^T P: those 8 tokens are what the B operand of one 32-token product wants from
//            the lane, if V^T takes tokens in the same order: lane l loads the 8 tokens' rows, at columns of its
//            own (l % 16), as whole vectors; operand e pairs up their e-th values, one v_perm per two.
// P goes into the product as the sum of two 16-bit numbers (three for fp32 queries over 8-bit pages), because its
// rounding to one would be as large an error as the rounding of the result.  fp32 pages use the fp32 MFMA.
// 8-bit codes are exact in bf16 and fp16; a row's scale multiplies its score, or its weight in P.
//
// Work is split over waves, over workgroups and joined with the usual weights exp(m_part - m): waves of a
// workgroup through LDS, workgroups through a workspace and a second kernel.
#include <algorithm>

#include "wc_paged.h"

namespace wc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 32;          // tokens a wave takes at a time

struct Paged {
  PagedTable t;
  const char *k, *v, *q;
  const float *ks, *vs;
  char* o;
  float* part;               // [seqs * heads][splits][dh]
  float2* ml;                // [seqs * heads][splits]: maximum and sum, a sum of -1 where there are no tokens
  const int32_t *lengths, *first;
  int64_t qn, qb, qh;
  int32_t heads, group, qtiles, splits, dh, row_bytes, most;
  FastDiv by_split, by_qtile, by_kvh, by_b;
  float scale;               // of the scores, times log2 e
};

// exp2 of a difference of scores; a part that holds nothing has m = -infinity
__device__ __forceinline__ float weight2(float m, float top) { return exp2f(m - top); }
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
__device__ __forceinline__ float byte_f32(uint32_t v, int i) { return static_cast<float>(static_cast<int8_t>(v >> (8 * i))); }

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

// 8 weights >= 0 as two planes, both over 0 where the weight is: the first is what 16 bits hold of a value just under
// the weight, so that an infinite value in V takes the sum to its infinity and not, by 0 or the other sign, to NaN.
template <typename MT>
__device__ __forceinline__ void weight_planes(const float (&p)[8], u32x4 (&out)[2]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = p[2 * e], b = p[2 * e + 1], under = 0x1.fffffep-1f;
    uint32_t w;
    if constexpr (std::is_same<MT, f16>::value)
      w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a * under, b * under));
    else
      w = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b * under), __builtin_bit_cast(uint32_t, a * under), 0x07060302u);
    out[0][e] = w;
    out[1][e] = pack2<MT>(a - unpack_lo<MT>(w), b - unpack_hi<MT>(w));
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

// QT: type of q and o; KT: stored type (int8_t for codes); DC: columns provided for; NW: waves
template <typename QT, typename KT, int DC, int NW>
__global__ __launch_bounds__(NW * 64) void paged_attention_kernel(Paged a) {
  constexpr bool kF32 = std::is_same<KT, float>::value;
  constexpr bool kQ8 = std::is_same<KT, int8_t>::value;
  // fp16 has no room for a weight times a row's scale: over codes, fp16 queries go as two bf16 planes
  typedef typename std::conditional<std::is_same<QT, f16>::value && !kQ8, f16, bf16>::type MT;
  constexpr int ES = sizeof(KT);
  constexpr int CH = 16 / ES;                                   // columns in 16 bytes
  constexpr int NCK = DC / (4 * CH);                            // 16-byte pieces of a K row per lane
  constexpr int VE = DC / 16, CE = VE * ES > 16 ? CH : VE, NCV = VE / CE;   // columns of V per lane
  constexpr int NF = DC / 32;                                   // 16-bit score products per 16 tokens
  constexpr int NQ = std::is_same<QT, float>::value ? 3 : std::is_same<QT, MT>::value ? 1 : 2;   // planes of q
  constexpr int NP = std::is_same<QT, float>::value ? 3 : 2;                                    // and of P
  // fp16 weights are taken 2^14 times as large (m - 14 in their exponents), so that those far under 1 keep their bits
  constexpr float kShift = std::is_same<MT, f16>::value ? 14.f : 0.f;
  typedef typename Raw<CE * ES>::type VR;
  extern __shared__ float lds[];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  uint32_t id = blockIdx.x;
  uint32_t up = fdiv(id, a.by_split);
  const int split = id - up * a.by_split.d;
  id = up;
  up = fdiv(id, a.by_qtile);
  const int qtile = id - up * a.by_qtile.d;
  id = up;
  const uint32_t seq = fdiv(id, a.by_kvh);
  const int kvh = id - seq * a.by_kvh.d;
  const uint32_t model = fdiv(seq, a.by_b), b = seq - model * a.by_b.d;
  const int gq = min(16, a.group - qtile * 16);                 // query heads of this workgroup
  const int head0 = kvh * a.group + qtile * 16;

  int hi = a.lengths[seq];
  if (hi > a.most) {
    hi = a.most;
    if (threadIdx.x == 0) paged_fault(a.t);
  }
  const int seq_lo = a.first ? max(a.first[seq], 0) : 0;
  // this workgroup's share: whole tiles, counted from the tile that holds the first token
  const int base = seq_lo & ~(kTile - 1);
  const int tiles = hi > seq_lo ? (hi - base + kTile - 1) / kTile : 0;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int tile_lo = split * per, tile_hi = min(tiles, tile_lo + per);

  // q: the same columns of each product as K's
  u32x4 qf[kF32 ? 1 : NF][NQ];
  float q32[kF32 ? NCK : 1][4];
  {
    const QT* q = reinterpret_cast<const QT*>(a.q) + model * a.qn + b * a.qb + (head0 + min(j, gq - 1)) * a.qh;
    if constexpr (kF32) {
#pragma unroll
      for (int c = 0; c < NCK; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = (c * 4 + g) * 4 + e;
          q32[c][e] = j < gq && d < a.dh ? to_f32(q[d]) : 0.f;
        }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = kQ8 ? ((f / 2) * 4 + g) * 16 + (f % 2) * 8 + e : (f * 4 + g) * 8 + e;
          x[e] = j < gq && d < a.dh ? to_f32(q[d]) : 0.f;
        }
        planes<MT, NQ>(x, qf[f]);
      }
    }
  }

  f32x4 acc[NCV][CE] = {};
  float m = -INFINITY, l = 0.f;
  bool any = false;

  // the pool's row of token `lane % 32` of a tile, -1 for none
  auto look = [&](int tile) {
    const int tok = base + tile * kTile + (lane & 31);
    int row = -1;
    if (tile < tile_hi && tok >= seq_lo && tok < hi) {
      row = paged_row(a.t, seq, tok, kvh);
      if (row < 0) paged_fault(a.t);
    }
    return row;
  };

  int row = look(tile_lo + wave);
  for (int tile = tile_lo + wave; tile < tile_hi; tile += NW) {
    const int next = look(tile + NW);
    const bool full = __all(row >= 0);
    any |= __any(row >= 0);
    // rows that no token has are read as row 0 of the pool and taken out afterwards
    float ks = 0.f, vs = 0.f;
    if constexpr (kQ8) {
      ks = row >= 0 ? a.ks[row] : 0.f;
      vs = row >= 0 ? a.vs[row] : 0.f;
    }
    u32x4 kf[2][NCK];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p = a.k + static_cast<int64_t>(max(__shfl(row, s * 16 + j, 64), 0)) * a.row_bytes;
#pragma unroll
      for (int c = 0; c < NCK; ++c) {
        const int at = (c * 4 + g) * 16;
        kf[s][c] = *reinterpret_cast<const u32x4*>(p + (at < a.row_bytes ? at : 0));
      }
    }
    int vrow[8];
    VR vf[8][NCV];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      vrow[u] = __shfl(row, (u >> 2) * 16 + g * 4 + (u & 3), 64);
      const char* p = a.v + static_cast<int64_t>(max(vrow[u], 0)) * a.row_bytes;
#pragma unroll
      for (int c = 0; c < NCV; ++c) {
        const int at = (c * 16 + j) * CE * ES;
        vf[u][c] = *reinterpret_cast<const VR*>(p + (at < a.row_bytes ? at : 0));
      }
    }
    // columns that a row doesn't have (their q is 0, but 0 times what stands elsewhere may not be)
    if (a.row_bytes < DC * ES) {
#pragma unroll
      for (int c = 0; c < NCK; ++c)
        if ((c * 4 + g) * 16 >= a.row_bytes) clear(kf[0][c]), clear(kf[1][c]);
    }

    f32x4 s2[2] = {};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if constexpr (kF32) {
#pragma unroll
        for (int c = 0; c < NCK; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s2[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, kf[s][c])[e], q32[c][e], s2[s], 0, 0, 0);
      } else {
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          u32x4 x;
          if constexpr (kQ8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t w = kf[s][f / 2][(f % 2) * 2 + e / 2];
              x[e] = pack2<MT>(byte_f32(w, (e & 1) * 2), byte_f32(w, (e & 1) * 2 + 1));
            }
          } else {
            x = kf[s][f];
          }
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n)
            s2[s] = mma16<MT>(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, qf[f][n]), s2[s]);
        }
      }
    }

    float p[8], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      p[u] = s2[u >> 2][u & 3] * a.scale;
      if constexpr (kQ8) p[u] *= __shfl(ks, (u >> 2) * 16 + g * 4 + (u & 3), 64);
      if (!full && vrow[u] < 0) p[u] = -INFINITY;
      top = fmaxf(top, p[u]);
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mn = fmaxf(m, top), shrink = weight2(m, finite_top(mn)), use = finite_top(mn) - kShift;
    m = mn;
    l *= shrink;
#pragma unroll
    for (int c = 0; c < NCV; ++c)
#pragma unroll
      for (int e = 0; e < CE; ++e) acc[c][e] *= shrink;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      p[u] = exp2f(p[u] - use);
      l += p[u];
      if constexpr (kQ8) p[u] *= __shfl(vs, (u >> 2) * 16 + g * 4 + (u & 3), 64);
    }
    if (!full) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (vrow[u] < 0) {
          p[u] = 0.f;
#pragma unroll
          for (int c = 0; c < NCV; ++c) clear(vf[u][c]);
        }
    }
    if constexpr (kF32) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int c = 0; c < NCV; ++c)
#pragma unroll
          for (int e = 0; e < CE; ++e)
            acc[c][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, dword(vf[u][c], e)), p[u], acc[c][e], 0, 0, 0);
    } else {
      u32x4 pf[NP];
      if constexpr (NP == 2)
        weight_planes<MT>(p, pf);
      else
        planes<MT, NP>(p, pf);
#pragma unroll
      for (int c = 0; c < NCV; ++c)
#pragma unroll
        for (int e = 0; e < CE; ++e) {
          u32x4 x;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if constexpr (kQ8)
              x[u] = pack2<MT>(byte_f32(dword(vf[2 * u][c], e / 4), e & 3), byte_f32(dword(vf[2 * u + 1][c], e / 4), e & 3));
            else
              x[u] = __builtin_amdgcn_perm(dword(vf[2 * u + 1][c], e / 2), dword(vf[2 * u][c], e / 2),
                                           e & 1 ? 0x07060302u : 0x05040100u);
          }
#pragma unroll
          for (int n = NP - 1; n >= 0; --n)
            acc[c][e] = mma16<MT>(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, pf[n]), acc[c][e]);
        }
    }
    row = next;
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // join the waves: [NW][gq][DC] outputs, then [NW][gq] maxima and sums (a sum of -1: no tokens)
  float* om = lds + NW * gq * DC;
  float* ol = om + NW * gq;
  if (j < gq) {
    float* o = lds + (wave * gq + j) * DC;
#pragma unroll
    for (int c = 0; c < NCV; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < CE; ++e) o[(c * 16 + g * 4 + r) * CE + e] = acc[c][e][r];
    if (g == 0) {
      om[wave * gq + j] = m;
      ol[wave * gq + j] = any ? l : -1.f;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < gq * DC; i += NW * 64) {
    const int h = i / DC, d = i - h * DC;
    float top = -INFINITY;
    for (int w = 0; w < NW; ++w) top = fmaxf(top, om[w * gq + h]);
    const float use = finite_top(top);
    float sum = 0.f, o = 0.f;
    bool some = false;
    for (int w = 0; w < NW; ++w) {
      const float lw = ol[w * gq + h];
      if (lw < 0.f) continue;
      some = true;
      const float f = weight2(om[w * gq + h], use);
      sum += f * lw;
      o += f * lds[(w * gq + h) * DC + d];
    }
    if (d >= a.dh) continue;
    const int64_t at = static_cast<int64_t>(seq) * a.heads + head0 + h;
    if (a.splits == 1) {
      reinterpret_cast<QT*>(a.o)[at * a.dh + d] = from_f32<QT>(some ? o / sum : 0.f);
    } else {
      a.part[(at * a.splits + split) * a.dh + d] = o;
      if (d == 0) a.ml[at * a.splits + split] = make_float2(top, some ? sum : -1.f);
    }
  }
}

// Joins the workgroups' parts of one (sequence, query head).
template <typename QT>
__global__ __launch_bounds__(256) void paged_join_kernel(const float* part, const float2* parts, int splits, int dh, QT* out) {
  const int64_t at = blockIdx.x;
  const float2* ml = parts + at * splits;
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s].x);
  const float use = finite_top(top);
  float sum = 0.f;
  bool some = false;
  for (int s = 0; s < splits; ++s) {
    const float2 x = ml[s];
    if (x.y < 0.f) continue;
    some = true;
    sum += weight2(x.x, use) * x.y;
  }
  for (int d = threadIdx.x; d < dh; d += 256) {
    float o = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float2 x = ml[s];
      if (x.y < 0.f) continue;
      o += weight2(x.x, use) * part[(at * splits + s) * dh + d];
    }
    out[at * dh + d] = from_f32<QT>(some ? o / sum : 0.f);
  }
}

// Workgroups a sequence's key head is split over: enough of them for the machine to have three in every compute
// unit, but none with less than a tile per wave.
constexpr int kWaves = 4;
int64_t splits_of(const wc_paged_attn_args& p) {
  const int64_t group = p.q_heads / p.cache.heads;
  const int64_t wgs = p.cache.n * p.cache.b * p.cache.heads * cdiv(group, 16);
  const int64_t most = cdiv(std::min(p.max_length, p.cache.table_len * p.cache.page_size), kWaves * kTile);
  return std::max<int64_t>(1, std::min({cdiv(768, wgs), most, int64_t(64)}));
}

template <typename QT, typename KT, int DC>
void launch(const Paged& a, int64_t grid, hipStream_t s) {
  const int gq = std::min(a.group, 16);
  const size_t lds = static_cast<size_t>(kWaves) * gq * (DC + 2) * sizeof(float);
  const auto kernel = paged_attention_kernel<QT, KT, DC, kWaves>;
  if (lds > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
  kernel<<<static_cast<uint32_t>(grid), kWaves * 64, lds, s>>>(a);
}

template <typename QT>
void dispatch(const Paged& a, bool q8, int64_t grid, hipStream_t s) {
  auto go = [&](auto k) {
    typedef decltype(k) KT;
    if (a.dh <= 64)
      launch<QT, KT, 64>(a, grid, s);
    else if (a.dh <= 128)
      launch<QT, KT, 128>(a, grid, s);
    else
      launch<QT, KT, 256>(a, grid, s);
  };
  if (q8)
    go(int8_t());
  else
    go(QT());
}

int32_t check(const wc_paged_attn_args& p, const char* what) {
  const wc_paged_cache& c = p.cache;
  if (int32_t rc = paged_check(c, what)) return rc;
  WC_REQUIRE(p.q_heads >= 0 && p.max_length >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(c.heads > 0 ? p.q_heads % c.heads == 0 : p.q_heads == 0, WC_ERR_SHAPE, "%s: %lld query heads over %lld key heads", what,
             (long long)p.q_heads, (long long)c.heads);
  WC_REQUIRE(p.q_heads <= 65535 && p.max_length < (1ll << 31) - 64, WC_ERR_LIMIT, "%s: more than 65535 heads or 2^31 tokens", what);
  // a launch holds fewer than 2^32 threads
  WC_REQUIRE(mul_sat({c.n, c.b, p.q_heads}) < (1ll << 23), WC_ERR_LIMIT, "%s: 2^23 rows or more", what);
  WC_REQUIRE(c.row * paged_es(c) <= 1024, WC_ERR_LIMIT, "%s: rows above 1024 bytes", what);
  return WC_OK;
}

}  // namespace
}  // namespace wc

extern "C" int64_t wc_paged_attention_workspace_bytes(const wc_paged_attn_args* args) {
  using namespace wc;
  clear_error();
  if (!args) {
    set_error(WC_ERR_NULL, "wc_paged_attention: null args");
    return -1;
  }
  if (check(*args, "wc_paged_attention")) return -1;
  if (args->cache.n == 0 || args->cache.b == 0 || args->q_heads == 0) return 0;
  const int64_t s = splits_of(*args);
  return s == 1 ? 0 : args->cache.n * args->cache.b * args->q_heads * s * (args->cache.head_dim + 2) * 4;
}

extern "C" int32_t wc_paged_attention(const wc_paged_attn_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_paged_attention";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_paged_attn_args& p = *args;
  const wc_paged_cache& c = p.cache;
  if (int32_t rc = check(p, what)) return rc;
  const int64_t seqs = c.n * c.b;
  if (seqs == 0 || p.q_heads == 0) return WC_OK;
  if (int32_t rc = paged_check_pointers(c, what)) return rc;
  const int es = dtype_size(c.dtype);
  WC_REQUIRE(p.q && p.o && p.lengths, WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(aligned(p.q, es) && aligned(p.o, es) && aligned(p.lengths, 4) && aligned(p.first, 4), WC_ERR_ALIGN,
             "%s: pointers must be aligned to their elements", what);
  Paged a;
  a.t = paged_table(c);
  a.k = static_cast<const char*>(c.k_pages);
  a.v = static_cast<const char*>(c.v_pages);
  a.ks = c.k_scales;
  a.vs = c.v_scales;
  a.q = static_cast<const char*>(p.q);
  a.o = static_cast<char*>(p.o);
  a.lengths = p.lengths;
  a.first = p.first;
  a.qn = p.q_stride_n;
  a.qb = p.q_stride_b;
  a.qh = p.q_stride_h;
  a.heads = static_cast<int32_t>(p.q_heads);
  a.group = static_cast<int32_t>(p.q_heads / c.heads);
  a.qtiles = static_cast<int32_t>(cdiv(a.group, 16));
  a.dh = static_cast<int32_t>(c.head_dim);
  a.row_bytes = static_cast<int32_t>(c.row * paged_es(c));
  a.most = static_cast<int32_t>(c.pages ? p.max_length : 0);      // a pool without pages has no row 0 either
  a.scale = p.scale * kLog2e;
  const int64_t splits = splits_of(p);
  a.splits = static_cast<int32_t>(splits);
  const int64_t need = splits == 1 ? 0 : seqs * p.q_heads * splits * (c.head_dim + 2) * 4;
  WC_REQUIRE(need == 0 || (p.workspace && p.workspace_bytes >= need), WC_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what,
             (long long)p.workspace_bytes, (long long)need);
  WC_REQUIRE(need == 0 || aligned(p.workspace, 16), WC_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  a.ml = static_cast<float2*>(p.workspace);
  a.part = need ? static_cast<float*>(p.workspace) + 2 * seqs * p.q_heads * splits : nullptr;
  a.by_split = make_fastdiv(static_cast<uint32_t>(splits));
  a.by_qtile = make_fastdiv(static_cast<uint32_t>(a.qtiles));
  a.by_kvh = make_fastdiv(static_cast<uint32_t>(c.heads));
  a.by_b = make_fastdiv(static_cast<uint32_t>(c.b));
  const int64_t grid = seqs * c.heads * a.qtiles * splits;
  const hipStream_t s = as_stream(stream);
  auto go = [&](auto t) {
    typedef decltype(t) QT;
    dispatch<QT>(a, c.bits == 8, grid, s);
    if (splits > 1)
      paged_join_kernel<QT><<<static_cast<uint32_t>(seqs * p.q_heads), 256, 0, s>>>(a.part, a.ml, a.splits, a.dh,
                                                                                 reinterpret_cast<QT*>(a.o));
  };
  if (c.dtype == WC_F32)
    go(float());
  else if (c.dtype == WC_BF16)
    go(bf16());
  else
    go(f16());
  return check_launch(what);
}
