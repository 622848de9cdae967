// Attention of one new token of every sequence over a prefix that groups of sequences share and over tokens of its own.
//
//   o = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),   s_i = scale q . k_i,   i over the prefix and the own tokens
//
// The softmax is joined from parts that have a maximum, a sum and an output each, so a prefix is walked once for all
// its sequences: their query heads are the rows that every K and V row meets, 16 for each tile of the matrix instructions.
// Both walks are one kernel, of stretches of tokens with rows that read them: a prefix with the heads of its sequences,
// and a sequence's own tokens with its heads.  A second kernel joins the parts.  Prefixes that more than 32 rows read in 16 bits
// are walked by shared_stream.hip instead.
//
// A wave takes 32 tokens at a time, K and V straight from memory into the operands of MFMAs:
//   scores   S [token][row] = K Q^T, lane l brings 16-byte pieces of token l % 16
//   softmax  the accumulator has row l % 16 and tokens 4 (l / 16) + r, of two tiles of 16 tokens
//   output   O^T [column][row] = V^T P, lane l loads those 8 tokens' rows at columns of its own, and operand e pairs
//            up their e-th values
//
// Own tokens are bound by memory and by waves that wait for their sequence's rows: 128 sequences of up to 500 tokens, 8 key heads of 128
// columns in bf16, 164 MB in 37 us (4.4 TB/s); 64 of up to 2000, 325 MB in 67 us (4.9 TB/s).  Small calls are bound by two launches and
// four waits for memory: 2 sequences over a prefix of 300 tokens 10.2 us.
#include <algorithm>

#include "wc_shared.h"

namespace wc {
namespace {

// Tiles of 32 tokens in a share at least (one prefix of 300 tokens, 3 x 3 of up to 1777, own tokens up to 2000: 1: 10.0, 27.9 and 42.2 us,
// 2: 10.2, 27.9 and 38.1, 4: 10.6, 29.6 and 38.7)
constexpr int kLeast = 2;

// QT: type of q and o; KT: stored type (int8_t for codes); DC: columns provided for; RT: tiles of 16 rows
template <typename QT, typename KT, int DC, int RT>
__device__ __forceinline__ void walk(const SharedAttn& a, const SharedWalk w, uint32_t id, float* lds) {
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
  constexpr int NP = std::is_same<MT, f16>::value ? 2 : 3;                                      // and of P
  // fp16 weights are taken 2^14 times as large (m - 14 in their exponents), so that those far under 1 keep their bits
  constexpr float kShift = std::is_same<MT, f16>::value ? 14.f : 0.f;
  constexpr int NW = kSharedWaves;
  typedef typename Raw<CE * ES>::type VR;

  const int lane0 = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t up = fdiv(id, w.by_tiles);
  const int row0 = (id - up * w.by_tiles.d) * (RT * 16);
  id = up;
  up = fdiv(id, a.by_kvh);
  const int kvh = id - up * a.by_kvh.d;
  // this workgroup's tiles: those of one unit, or a share of the line
  int unit = up, start = 0, from = 0, to = 1 << 30;
  if (w.budget > 0) {
    const SharedLine line = shared_line(w, lane0);
    if (id == 0 && row0 == 0 && wave == 0) shared_list(w, line.size, lane0);
    from = up * line.size;
    if (from >= line.total) return;
    to = min(from + line.size, line.total);
    const int2 first = shared_find(w, from, lane0);
    unit = first.x;
    start = first.y;
  }
  for (;; ++unit) {
    // What depends on the lane and the sizes alone would be kept from one unit to the next, in more registers than there
    // are; it is worked out again.
    int lane = lane0, rows = w.rows, dh = a.dh;
    asm volatile("" : "+v"(lane), "+s"(rows), "+s"(dh));
    const int j = lane & 15, g = lane >> 4;
    const uint32_t model = fdiv(unit, w.by_units), b0 = (unit - model * w.by_units.d) * w.share;
    const int tile_lo = max(from - start, 0);
    // The table's entry for token `lane % 32` of a tile, two tiles ahead of its use; nothing looks at it (and so waits for
    // it) before row_of, the pool's row of that token or -1 for none.
    auto look = [&](int tile) { return paged_entry(w.t, unit, static_cast<uint32_t>(tile) * kPagedTile + (lane & 31)); };
    int row = look(tile_lo + wave), next = look(tile_lo + wave + NW);
    // The rows of q: row r is head r % group of sequence r / group; past the last the last again, from column 0 instead of not
    // at all, without branches that every load would wait in.  What these loads, the length and the table's entries depend on is the
    // unit alone, so that one wait serves them all.
    constexpr int N = kF32 ? 4 : 8, NX = kF32 ? NCK : NF;
    auto column = [&](int i) {                                    // the same columns of each product as K's
      return kF32 ? (i * 4 + g) * 4 : kQ8 ? ((i / 2) * 4 + g) * 16 + (i % 2) * 8 : (i * 4 + g) * 8;
    };
    constexpr int NV = 16 / sizeof(QT);
    u32x4 raw[RT][NX][N / NV];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = min(row0 + t * 16 + j, rows - 1);
      const uint32_t s = fdiv(r, a.by_group), h = r - s * a.by_group.d;
      const QT* q = reinterpret_cast<const QT*>(a.q) + model * a.qn + (b0 + s) * a.qb + (kvh * a.group + h) * a.qh;
#pragma unroll
      for (int i = 0; i < NX * N / NV; ++i) {
        const int d = column(i / (N / NV)) + i % (N / NV) * NV;
        u32x4& x = raw[t][i / (N / NV)][i % (N / NV)];
        if (a.qvec) {
          x = *reinterpret_cast<const u32x4*>(q + (d < dh ? d : 0));
        } else {
          QT v[NV];
#pragma unroll
          for (int e = 0; e < NV; ++e) v[e] = q[d + e < dh ? d + e : 0];
          __builtin_memcpy(&x, v, sizeof v);
        }
      }
    }
    const PagedSpan span = shared_span(w, unit);
    const int hi = span.hi, tiles = paged_tiles(span), tile_hi = min(tiles, to - start);
    if (w.budget == 0 && span.cut && threadIdx.x == 0) paged_fault(w.t);
    start += tiles;
    if (w.budget > 0 && tile_lo >= tile_hi) continue;             // a unit without tokens
    u32x4 qf[RT][kF32 ? 1 : NF][NQ];
    float q32[RT][kF32 ? NCK : 1][4];

    f32x4 acc[RT][NCV][CE] = {};
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) m[t] = -INFINITY, l[t] = 0.f;
    bool any = false;

    auto row_of = [&](int tile, int page) {
      const int tok = tile * kPagedTile + (lane & 31);
      if (tile >= tile_hi || tok >= hi) return -1;
      const int r = paged_row(w.t, page, tok, kvh);
      if (r < 0) paged_fault(w.t);
      return r;
    };
    // Rows that no token has are read as row 0 of the pool and taken out afterwards.  K comes one tile ahead, into the
    // registers that the scores have just been taken from, while softmax and V keep the wave busy.
    u32x4 kf[2][NCK];
    float ks = 0.f;
    auto load_k = [&](int row) {
      if constexpr (kQ8) ks = a.ks[max(row, 0)];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const char* p = a.k + static_cast<int64_t>(max(__shfl(row, s * 16 + j, 64), 0)) * a.row_bytes;
#pragma unroll
        for (int c = 0; c < NCK; ++c) {
          const int at = (c * 4 + g) * 16;
          kf[s][c] = *reinterpret_cast<const u32x4*>(p + (at < a.row_bytes ? at : 0));
        }
      }
    };
    if (tile_lo + wave < tile_hi) {
      row = row_of(tile_lo + wave, row);
      load_k(row);
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < NX; ++i) {
          QT v[N];
          float x[N];
          __builtin_memcpy(v, raw[t][i], sizeof v);
#pragma unroll
          for (int e = 0; e < N; ++e) x[e] = column(i) + e < dh ? to_f32(v[e]) : 0.f;
          if constexpr (kF32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) q32[t][i][e] = x[e];
          } else {
            planes<MT, NQ>(x, qf[t][i]);
          }
        }
    }
    for (int tile = tile_lo + wave; tile < tile_hi; tile += NW) {
      const bool full = __all(row >= 0);
      any |= __any(row >= 0);
      float vs = 0.f;
      if constexpr (kQ8) vs = a.vs[max(row, 0)];
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

      f32x4 s2[RT][2] = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if constexpr (kF32) {
#pragma unroll
          for (int c = 0; c < NCK; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int t = 0; t < RT; ++t)
                s2[t][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, kf[s][c])[e], q32[t][c][e], s2[t][s], 0, 0, 0);
        } else {
#pragma unroll
          for (int f = 0; f < NF; ++f) {
            u32x4 x;
            if constexpr (kQ8) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t c = kf[s][f / 2][(f % 2) * 2 + e / 2];
                x[e] = pack2<MT>(byte_f32(c, (e & 1) * 2), byte_f32(c, (e & 1) * 2 + 1));
              }
            } else {
              x = kf[s][f];
            }
#pragma unroll
            for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
              for (int t = 0; t < RT; ++t)
                s2[t][s] = mma16<MT>(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, qf[t][f][n]), s2[t][s]);
          }
        }
      }
      float kscale[kQ8 ? 8 : 1], vscale[kQ8 ? 8 : 1];
      if constexpr (kQ8) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          kscale[u] = __shfl(ks, (u >> 2) * 16 + g * 4 + (u & 3), 64);
          vscale[u] = __shfl(vs, (u >> 2) * 16 + g * 4 + (u & 3), 64);
        }
      }
      // behind the last tile too (as row 0): were there a way round these loads, the wait for V would have to be one for
      // everything in flight
      row = row_of(tile + NW, next);
      load_k(row);
      next = look(tile + 2 * NW);
      u32x4 pf[RT][NP];
      float p[RT][8];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          p[t][u] = s2[t][u >> 2][u & 3] * a.scale;
          if constexpr (kQ8) p[t][u] *= kscale[u];
          if (!full && vrow[u] < 0) p[t][u] = -INFINITY;
          top = fmaxf(top, p[t][u]);
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float mn = fmaxf(m[t], top), use = finite_top(mn) - kShift;
        const float shrink = weight2(m[t], finite_top(mn));
        m[t] = mn;
        l[t] *= shrink;
#pragma unroll
        for (int c = 0; c < NCV; ++c)
#pragma unroll
          for (int e = 0; e < CE; ++e) acc[t][c][e] *= shrink;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          p[t][u] = __builtin_amdgcn_exp2f(p[t][u] - use);
          l[t] += p[t][u];
          if constexpr (kQ8) p[t][u] *= vscale[u];
        }
      }
      if (!full) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (vrow[u] < 0) {
#pragma unroll
            for (int t = 0; t < RT; ++t) p[t][u] = 0.f;
#pragma unroll
            for (int c = 0; c < NCV; ++c) clear(vf[u][c]);
          }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        if constexpr (!kF32) {
          if constexpr (std::is_same<QT, float>::value)
            planes<MT, NP>(p[t], pf[t]);
          else
            weight_planes<MT, NP>(p[t], pf[t]);
        }
      }
      if constexpr (kF32) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int c = 0; c < NCV; ++c)
#pragma unroll
            for (int e = 0; e < CE; ++e)
#pragma unroll
              for (int t = 0; t < RT; ++t)
                acc[t][c][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, dword(vf[u][c], e)), p[t][u], acc[t][c][e], 0, 0, 0);
      } else {
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
#pragma unroll
              for (int t = 0; t < RT; ++t)
                acc[t][c][e] = mma16<MT>(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, pf[t][n]), acc[t][c][e]);
          }
      }
    }

    // Join the waves, a tile of rows at a time: [NW][16][kRow] outputs (rows 4 values apart from whole banks: with rows of DC the
    // 16 that a wave writes at a time all meet in one bank, 10 us of 41 over 128 sequences of up to 500 tokens), then [NW][16] maxima and
    // sums (a sum of -1: no tokens),
    // which become the weights of the waves' outputs
    constexpr int kRow = DC + 4;
    float* om = lds + NW * 16 * kRow;
    float* ol = om + NW * 16;
    const int64_t first = static_cast<int64_t>(w.budget > 0 ? up + unit : unit) * w.share;      // part's first (sequence, ..)
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (row0 + t * 16 >= rows) break;
      l[t] += __shfl_xor(l[t], 16, 64);
      l[t] += __shfl_xor(l[t], 32, 64);
      __syncthreads();
      if (j < rows - row0 - t * 16) {
        float* o = lds + (wave * 16 + j) * kRow;
#pragma unroll
        for (int c = 0; c < NCV; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < CE; ++e) o[(c * 16 + g * 4 + r) * CE + e] = acc[t][c][e][r];
        if (g == 0) {
          om[wave * 16 + j] = m[t];
          ol[wave * 16 + j] = any ? l[t] : -1.f;
        }
      }
      __syncthreads();
      auto at = [&](int h) {                         // of row h of the tile: its place among the part's (sequence, head)
        const uint32_t r = row0 + t * 16 + h, s = fdiv(r, a.by_group);
        return (first + s) * a.heads + kvh * a.group + (r - s * a.by_group.d);
      };
      if (static_cast<int>(threadIdx.x) < min(16, rows - row0 - t * 16)) {
        const int h = threadIdx.x;
        float mw[NW], lw[NW], top = -INFINITY, sum = 0.f;
        bool some = false;
#pragma unroll
        for (int v = 0; v < NW; ++v) {
          mw[v] = om[v * 16 + h];
          lw[v] = ol[v * 16 + h];
          top = fmaxf(top, mw[v]);
          some |= !(lw[v] < 0.f);
        }
#pragma unroll
        for (int v = 0; v < NW; ++v) {
          const float f = weight2(mw[v], finite_top(top));            // 0 for a wave without tokens
          om[v * 16 + h] = f;
          sum += lw[v] < 0.f ? 0.f : f * lw[v];
        }
        w.ml[at(h)] = make_float2(top, some ? sum : -1.f);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < min(16, rows - row0 - t * 16) * (DC / 4); i += NW * 64) {
        const int h = i / (DC / 4), d = i % (DC / 4) * 4;
        f32x4 sum = {};
#pragma unroll
        for (int v = 0; v < NW; ++v) sum += om[v * 16 + h] * *reinterpret_cast<const f32x4*>(lds + (v * 16 + h) * kRow + d);
        float* y = w.part + at(h) * dh;
        if (dh % 4 == 0) {
          if (d < dh) *reinterpret_cast<f32x4*>(y + d) = sum;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < dh) y[d + e] = sum[e];
        }
      }
    }
    if (w.budget == 0 || start >= to) return;
    __syncthreads();
  }
}

template <typename QT, typename KT, int DC, int RT>
__global__ __launch_bounds__(kSharedWaves * 64) void shared_attention_kernel(SharedAttn a) {
  extern __shared__ float lds[];
  const int own = static_cast<int>(blockIdx.x) >= a.blocks;
  const uint32_t id = blockIdx.x - (own ? a.blocks : 0);
  if constexpr (RT == 1) {
    const SharedWalk w = own ? a.walk[1] : a.walk[0];        // a copy: an index into the arguments would be followed with every use
    walk<QT, KT, DC, 1>(a, w, id, lds);
  } else {
    if (own)
      walk<QT, KT, DC, 1>(a, a.walk[1], id, lds);
    else
      walk<QT, KT, DC, RT>(a, a.walk[0], id, lds);
  }
}

// Joins the parts of a (sequence, query head), one wave for each: lane s has the weight of part s, 64 parts at a time, and
// as many parts as columns leave lanes for are added up side by side.  VEC: rows are whole vectors.
template <typename QT, bool VEC>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedAttn a, uint32_t total) {
  const int lane = threadIdx.x & 63;
  const uint32_t at = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (at >= total) return;
  const uint32_t seq = fdiv(at, a.by_heads), head = at - seq * a.by_heads.d;
  const uint32_t unit = fdiv(seq, a.by_share), place = seq - unit * a.by_share.d;
  const SharedWalk w0 = a.walk[0], w1 = a.walk[1];
  const int2 p0 = w0.budget > 0 ? w0.parts[unit] : make_int2(unit, 1), p1 = w1.budget > 0 ? w1.parts[seq] : make_int2(seq, 1);
  const int n0 = p0.y, n = w1.lengths[seq] < 0 ? 0 : n0 + p1.y;
  // row of part s of these: the prefix's, then the own
  auto row = [&](int s) {
    return s < n0 ? ((p0.x + s) * static_cast<int64_t>(w0.share) + place) * a.heads + head
                  : (p1.x + s - n0) * static_cast<int64_t>(a.heads) + head;
  };
  auto mass = [&](int s) { return s < n ? (s < n0 ? w0.ml : w1.ml)[row(s)] : make_float2(-INFINITY, -1.f); };
  const float2 first = mass(lane);
  float top = first.x;
  bool some = !(first.y < 0.f);
  for (int s = 64 + lane; s < n; s += 64) {
    const float2 x = mass(s);
    top = fmaxf(top, x.x);
    some |= !(x.y < 0.f);
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  some = __any(some);
  int lanes = 1;                                       // of a row: a power of two
  while (lanes * 4 < a.dh) lanes *= 2;
  const int q = lane & (lanes - 1), g = lane / lanes, groups = 64 / lanes;
  float sum = 0.f;
  f32x4 o = {};
  for (int s0 = 0; s0 < n; s0 += 64) {
    const float2 x = s0 ? mass(s0 + lane) : first;
    const float f = x.y < 0.f ? 0.f : weight2(x.x, finite_top(top));       // 0 for a part without tokens, which holds zeros
    sum += x.y < 0.f ? 0.f : f * x.y;
    const int m = min(64, n - s0);
    // eight outputs a lane on their way together; past the last part the last again, which is not added
    for (int i = g; i - g < m; i += 8 * groups) {
      f32x4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int c = s0 + min(i + u * groups, m - 1);
        const float* p = (c < n0 ? w0.part : w1.part) + row(c) * a.dh;
        if constexpr (VEC) {
          v[u] = *reinterpret_cast<const f32x4*>(p + (q * 4 < a.dh ? q * 4 : 0));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = p[q * 4 + e < a.dh ? q * 4 + e : 0];
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float weight = __shfl(f, min(i + u * groups, 63), 64);
        if (i + u * groups < m) o += weight * v[u];
      }
    }
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
  for (int off = lanes; off < 64; off *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off, 64);
  if (g) return;
  QT* y = reinterpret_cast<QT*>(a.o) + static_cast<int64_t>(at) * a.dh;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (q * 4 + e < a.dh) y[q * 4 + e] = from_f32<QT>(some ? o[e] / sum : 0.f);
}

// How the work is spread: tiles of 16 rows that a workgroup of the prefixes' walk has, and shares of both lines (own tokens
// 0: whole sequences)
struct Plan {
  int stream, rt;            // rows of a workgroup of the walk through LDS, or 0: tiles of 16 rows
  int64_t budget[2], parts[2];
};
int tiles_of_rows(const wc_shared_attn_args& p) {
  return p.share * (p.q_heads / p.cache.heads) <= 16 || (p.cache.head_dim > 128 && p.cache.dtype == WC_F32) ? 1 : 2;
}
Plan plan_of(const wc_shared_attn_args& p) {
  Plan plan;
  plan.stream = shared_stream_rows(p);
  plan.rt = plan.stream ? plan.stream / 16 : tiles_of_rows(p);
  const int64_t group = p.q_heads / p.cache.heads, units = p.cache.n * (p.cache.b / p.share), seqs = p.cache.n * p.cache.b;
  const int64_t heads0 = p.cache.heads * cdiv(p.share * group, plan.rt * 16), heads1 = p.cache.heads * cdiv(group, 16);
  // Workgroups of one round where a unit holds two, as it does in 16 bits of up to 128 columns (up to 256 registers; fewer of 64 columns, where it
  // would hold three).  fp32 of 128 columns and all of more than 128 (259 to 512 registers) take two rounds of one.
  const int64_t target = 512;
  plan.budget[0] = std::min<int64_t>(cdiv(target, heads0), kSharedTarget);
  plan.parts[0] = plan.budget[0] + units;
  // Sequences stay whole where they are short, or many for their length (45 of up to 130 tokens, 2 key heads: 29.6 us, cut 34.5; 128 of
  // up to 500, 8 key heads: 83.7 and 87.4); few long ones are cut (4 of up to 1000, 8 key heads: whole 17.5, cut 12.1).
  const bool whole = p.max_length <= 256 || seqs * heads1 >= (p.max_length <= 1024 ? 256 : 2048);
  plan.budget[1] = whole ? 0 : std::min<int64_t>(cdiv(target, heads1), kSharedTarget);
  plan.parts[1] = plan.budget[1] + seqs;
  return plan;
}
// outputs of both walks, their maxima and sums, the lists of parts
struct Space {
  int64_t part[2], ml[2], list[2], bytes;
};
Space space_of(const wc_shared_attn_args& p, const Plan& plan) {
  const int64_t units = p.cache.n * (p.cache.b / p.share), seqs = p.cache.n * p.cache.b;
  const int64_t rows[2] = {plan.parts[0] * p.share * p.q_heads, plan.parts[1] * p.q_heads};
  Space s;
  int64_t at = 0;
  for (int i = 0; i < 2; ++i) {
    s.part[i] = at;
    at += (rows[i] * p.cache.head_dim * 4 + 15) / 16 * 16;
  }
  for (int i = 0; i < 2; ++i) {
    s.ml[i] = at;
    at += rows[i] * 8;
  }
  s.list[0] = at;
  s.list[1] = at + units * 8;
  s.bytes = s.list[1] + seqs * 8;
  return s;
}

template <typename QT, typename KT, int DC, int RT>
void launch(const SharedAttn& a, int64_t grid, hipStream_t s) {
  constexpr size_t lds = static_cast<size_t>(kSharedWaves) * 16 * (DC + 6) * sizeof(float);
  const auto kernel = shared_attention_kernel<QT, KT, DC, RT>;
  if (lds > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
  kernel<<<static_cast<uint32_t>(grid), kSharedWaves * 64, lds, s>>>(a);
}

template <typename QT>
void dispatch(const SharedAttn& a, bool q8, int rt, int64_t grid, hipStream_t s) {
  auto go = [&](auto k, auto dc) {
    typedef decltype(k) KT;
    constexpr int DC = decltype(dc)::value;
    if (rt == 1) return launch<QT, KT, DC, 1>(a, grid, s);
    if constexpr (DC <= 128 || sizeof(QT) == 2) launch<QT, KT, DC, 2>(a, grid, s);
  };
  auto width = [&](auto k) {
    if (a.dh <= 64)
      go(k, std::integral_constant<int, 64>());
    else if (a.dh <= 128)
      go(k, std::integral_constant<int, 128>());
    else
      go(k, std::integral_constant<int, 256>());
  };
  if (q8)
    width(int8_t());
  else
    width(QT());
}

int64_t most_of(const wc_shared_attn_args& p, int i) {
  const int64_t len = i ? p.cache.table_len : p.prefix_len, most = i ? p.max_length : p.max_prefix;
  return p.cache.pages ? std::min(most, len * p.cache.page_size) : 0;
}

int32_t check(const wc_shared_attn_args& p, const char* what) {
  const wc_paged_cache& c = p.cache;
  if (int32_t rc = paged_check(c, what)) return rc;
  WC_REQUIRE(p.q_heads >= 0 && p.max_prefix >= 0 && p.max_length >= 0 && p.prefix_len >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(p.share > 0 && c.b % p.share == 0, WC_ERR_SHAPE, "%s: %lld sequences in groups of %lld", what, (long long)c.b, (long long)p.share);
  WC_REQUIRE(c.heads > 0 ? p.q_heads % c.heads == 0 : p.q_heads == 0, WC_ERR_SHAPE, "%s: %lld query heads over %lld key heads", what,
             (long long)p.q_heads, (long long)c.heads);
  WC_REQUIRE(p.q_heads <= 65535 && p.max_prefix < (1ll << 31) - 64 && p.max_length < (1ll << 31) - 64 && p.prefix_len < (1ll << 31),
             WC_ERR_LIMIT, "%s: more than 65535 heads or 2^31 tokens", what);
  WC_REQUIRE(p.prefix_len <= 1 || p.prefix_stride >= 0, WC_ERR_ARG, "%s: negative table stride", what);
  // a launch holds fewer than 2^32 threads, and counts tiles in 32 bits
  WC_REQUIRE(mul_sat({c.n, c.b, p.q_heads}) < (1ll << 22), WC_ERR_LIMIT, "%s: 2^22 rows or more", what);
  WC_REQUIRE(c.row * paged_es(c) <= 1024, WC_ERR_LIMIT, "%s: rows above 1024 bytes", what);
  WC_REQUIRE(paged_countable(c.n * (c.b / p.share), most_of(p, 0)) && paged_countable(c.n * c.b, most_of(p, 1)), WC_ERR_LIMIT,
             "%s: more than 2^35 tokens by the bounds", what);
  return WC_OK;
}

}  // namespace
}  // namespace wc

extern "C" int64_t wc_shared_attention_workspace_bytes(const wc_shared_attn_args* args) {
  using namespace wc;
  clear_error();
  if (!args) {
    set_error(WC_ERR_NULL, "wc_shared_attention: null args");
    return -1;
  }
  if (check(*args, "wc_shared_attention")) return -1;
  if (args->cache.n == 0 || args->cache.b == 0 || args->q_heads == 0) return 0;
  return space_of(*args, plan_of(*args)).bytes;
}

extern "C" int32_t wc_shared_attention(const wc_shared_attn_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_shared_attention";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_shared_attn_args& p = *args;
  const wc_paged_cache& c = p.cache;
  if (int32_t rc = check(p, what)) return rc;
  const int64_t seqs = c.n * c.b, units = seqs / p.share;
  if (seqs == 0 || p.q_heads == 0) return WC_OK;
  if (int32_t rc = paged_check_pointers(c, what)) return rc;
  const int es = dtype_size(c.dtype);
  WC_REQUIRE(p.q && p.o && p.lengths && p.prefix_lengths && (p.prefix_len == 0 || p.prefix_table), WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(aligned(p.q, es) && aligned(p.o, es) && aligned(p.lengths, 4) && aligned(p.prefix_lengths, 4) && aligned(p.prefix_table, 4),
             WC_ERR_ALIGN, "%s: pointers must be aligned to their elements", what);
  const Plan plan = plan_of(p);
  const Space space = space_of(p, plan);
  WC_REQUIRE(p.workspace && p.workspace_bytes >= space.bytes, WC_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what,
             (long long)p.workspace_bytes, (long long)space.bytes);
  WC_REQUIRE(aligned(p.workspace, 16), WC_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  SharedAttn a;
  a.k = static_cast<const char*>(c.k_pages);
  a.v = static_cast<const char*>(c.v_pages);
  a.ks = c.k_scales;
  a.vs = c.v_scales;
  a.q = static_cast<const char*>(p.q);
  a.o = static_cast<char*>(p.o);
  a.qn = p.q_stride_n;
  a.qb = p.q_stride_b;
  a.qh = p.q_stride_h;
  a.heads = static_cast<int32_t>(p.q_heads);
  a.group = static_cast<int32_t>(p.q_heads / c.heads);
  a.dh = static_cast<int32_t>(c.head_dim);
  a.row_bytes = static_cast<int32_t>(c.row * paged_es(c));
  a.qvec = c.head_dim * es % 16 == 0 && aligned(p.q, 16) && ubytes(p.q_stride_n, es) % 16 == 0 &&
           ubytes(p.q_stride_b, es) % 16 == 0 && ubytes(p.q_stride_h, es) % 16 == 0;
  a.scale = p.scale * kLog2e;
  a.by_kvh = make_fastdiv(static_cast<uint32_t>(c.heads));
  a.by_group = make_fastdiv(static_cast<uint32_t>(a.group));
  a.by_heads = make_fastdiv(static_cast<uint32_t>(a.heads));
  a.by_share = make_fastdiv(static_cast<uint32_t>(p.share));
  wc_paged_cache prefix = c;
  prefix.table = p.prefix_table;
  prefix.table_len = p.prefix_len;
  prefix.table_stride = p.prefix_stride;
  int64_t blocks[2];
  for (int i = 0; i < 2; ++i) {
    SharedWalk& w = a.walk[i];
    w.lengths = i ? p.lengths : p.prefix_lengths;
    w.t = paged_table(i ? c : prefix, w.lengths);
    char* ws = static_cast<char*>(p.workspace);
    w.part = reinterpret_cast<float*>(ws + space.part[i]);
    w.ml = reinterpret_cast<float2*>(ws + space.ml[i]);
    w.parts = reinterpret_cast<int2*>(ws + space.list[i]);
    w.units = static_cast<int32_t>(i ? seqs : units);
    w.share = static_cast<int32_t>(i ? 1 : p.share);
    w.budget = static_cast<int32_t>(plan.budget[i]);
    w.least = kLeast;
    w.most = static_cast<int32_t>(most_of(p, i));
    w.rows = w.share * a.group;
    const int64_t tiles = cdiv(w.rows, i ? 16 : plan.rt * 16);
    w.by_tiles = make_fastdiv(static_cast<uint32_t>(tiles));
    w.by_units = make_fastdiv(static_cast<uint32_t>(i ? c.b : c.b / p.share));
    blocks[i] = (w.budget ? w.budget : w.units) * c.heads * tiles;
  }
  a.blocks = static_cast<int32_t>(blocks[0]);
  const hipStream_t s = as_stream(stream);
  auto go = [&](auto t) {
    typedef decltype(t) QT;
    if (plan.stream) {
      shared_stream(a, c.dtype, c.bits == 8, plan.stream, blocks[0], s);
      a.blocks = 0;
      dispatch<QT>(a, c.bits == 8, 1, blocks[1], s);
    } else {
      dispatch<QT>(a, c.bits == 8, plan.rt, blocks[0] + blocks[1], s);
    }
    const uint32_t total = static_cast<uint32_t>(seqs * p.q_heads);
    (c.head_dim % 4 ? shared_join_kernel<QT, false> : shared_join_kernel<QT, true>)<<<(total + 3) / 4, 256, 0, s>>>(a, total);
  };
  if (c.dtype == WC_F32)
    go(float());
  else if (c.dtype == WC_BF16)
    go(bf16());
  else
    go(f16());
  return check_launch(what);
}
