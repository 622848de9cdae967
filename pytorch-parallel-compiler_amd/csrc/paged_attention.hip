// Attention of one new token of every sequence over its pages of cached keys and values.
//
//   o = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),   s_i = scale q . k_i,   m the running maximum
//
// in one pass over the sequence.  A query head group shares a key head, so up to 16 query heads are the columns of
// one MFMA tile and every K and V row is read once for all of them.  What bounds it is that reading: 4 flops per
// stored value and query head, far under the machine's balance.  The matrix instructions run mostly empty for small
// groups and in 16 bits still cost a tenth of the time their rows take to arrive.  32 query heads over 8 key heads of
// 128 columns: 2 sequences of 131072 and 32768 tokens in bf16 (671 MB) 121 us, 5.5 TB/s; 64 sequences of 1000 to 4000
// tokens in 8 bits (335 MB) 76 us, 4.4 TB/s, where turning codes into numbers takes half the instructions.
//
// A wave takes 32 tokens at a time, and nothing but the sum over its lanes ever leaves its registers:
//   scores   S [token][query] = K Q^T, K rows as the A operand: lane l brings 16-byte pieces of token l % 16, Q the
//            same columns, so the order of columns inside the product is free and pieces are whole vectors.
//   softmax  the accumulator has query l % 16 and tokens 4 (l / 16) + r, of two tiles of 16 tokens.
//   output   O^T [column][query] = V^T P: those 8 tokens are what the B operand of one 32-token product wants from
//            the lane, if V^T takes tokens in the same order: lane l loads the 8 tokens' rows, at columns of its
//            own (l % 16), as whole vectors; operand e pairs up their e-th values, one v_perm per two.
// P goes into the product as the sum of three bf16 numbers, or two fp16 ones: of two bf16 its last 2^-17 would be lost, which
// values that cancel show (and which moves 0.4 % of bf16 outputs by a step where fp32 sums move 0.1 %); the third costs
// nothing where memory bounds it and 3 % over codes.  fp32 pages use the fp32 MFMA.
// 8-bit codes are exact in bf16 and fp16; a row's scale multiplies its score, or its weight in P.
//
// Work is split over waves, over workgroups and joined with the usual weights exp(m_part - m): waves of a
// workgroup through LDS, workgroups through a workspace and a second kernel.
#include <algorithm>

#include "wc_paged_attn.h"

namespace wc {
namespace {

constexpr int kTile = kPagedTile;  // tokens a wave takes at a time
constexpr int kLeast = 8;          // tiles in a part at least, two for each of its waves (2 sequences of 2000 and 500 tokens:
                                   // 13.8 us; 4 tiles 13.4, 16 tiles 15.8; 8 of 3000 to 750: 22.3, 22.2, 21.1)
constexpr int kTarget = 1024;      // shares of the line at most

struct Paged {
  PagedTable t;
  const char *k, *v, *q;
  const float *ks, *vs;
  char* o;
  // parts, where sequences are split (budget > 0): [parts][heads][dh] outputs, [parts][heads] maximum and sum (-1 where
  // there are no tokens), and for each sequence its first part and how many it has
  float* part;
  float2* ml;
  int2* parts;
  const int32_t *lengths, *first;
  int64_t qn, qb, qh;
  int32_t seqs, heads, group, budget, dh, row_bytes, most, qvec;    // qvec: rows of q are whole 16-byte vectors
  FastDiv by_qtile, by_kvh, by_b;
  float scale;               // of the scores, times log2 e
};

__device__ __forceinline__ PagedSpan span_of(const Paged& a, int64_t seq) {
  return paged_span(a.first ? a.first[seq] : 0, a.lengths[seq], a.most);
}

// Where sequences are cut, the tiles of all of them count as one line, of which every workgroup (of a key head) has an
// equal share however uneven the lengths are: share w is tiles [w size, (w + 1) size), of one sequence or the ends
// and wholes of several.  What share w has of sequence s is part w + s: no two are alike, a sequence's parts are
// neighbours, and there are at most shares + sequences of them.  Every wave finds its share from the lengths by itself.
struct Line {
  int size, total;           // tiles in a share, in all
};
__device__ __forceinline__ Line line_of(const Paged& a, int lane) {
  int total = 0;
  for (int s = lane; s < a.seqs; s += 64) total += paged_tiles(span_of(a, s));
#pragma unroll
  for (int off = 32; off; off >>= 1) total += __shfl_xor(total, off, 64);
  return Line{max((total + a.budget - 1) / a.budget, kLeast), total};
}
// the sequence that has tile `at` of the line (at < total), and the line's tiles before it
__device__ __forceinline__ int2 find_tile(const Paged& a, int at, int lane) {
  int done = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    const int s = s0 + lane, n = s < a.seqs ? paged_tiles(span_of(a, s)) : 0;
    const int start = done + before(n, lane);
    const uint64_t mine = __ballot(at >= start && at < start + n);
    if (mine) {
      const int l = __ffsll(static_cast<unsigned long long>(mine)) - 1;
      return make_int2(s0 + l, __shfl(start, l, 64));
    }
    done = __shfl(start + n, 63, 64);
  }
  return make_int2(a.seqs, 0);
}
// each sequence's first part and how many it has, for the kernel that joins them; and the fault of lengths that were cut,
// of sequences without a tile (which no share visits) too
__device__ __forceinline__ void list_parts(const Paged& a, int size, int lane) {
  int done = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    const int s = s0 + lane;
    const PagedSpan span = s < a.seqs ? span_of(a, s) : PagedSpan{0, 0, false};
    if (span.cut) paged_fault(a.t);
    const int n = paged_tiles(span);
    const int start = done + before(n, lane), w0 = start / size;
    if (s < a.seqs) a.parts[s] = n ? make_int2(w0 + s, (start + n - 1) / size - w0 + 1) : make_int2(0, 0);
    done = __shfl(start + n, 63, 64);
  }
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
  constexpr int NP = std::is_same<MT, f16>::value ? 2 : 3;                                      // and of P
  // fp16 weights are taken 2^14 times as large (m - 14 in their exponents), so that those far under 1 keep their bits
  constexpr float kShift = std::is_same<MT, f16>::value ? 14.f : 0.f;
  typedef typename Raw<CE * ES>::type VR;
  extern __shared__ float lds[];

  const int lane0 = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t id = blockIdx.x;
  uint32_t up = fdiv(id, a.by_qtile);
  const int qtile = id - up * a.by_qtile.d;
  id = up;
  up = fdiv(id, a.by_kvh);
  const int kvh = id - up * a.by_kvh.d;
  const int gq0 = min(16, a.group - qtile * 16);                // query heads of this workgroup
  const int head0 = kvh * a.group + qtile * 16;
  // this workgroup's tiles: those of one sequence, or a share of the line
  int seq = up, start = 0, from = 0, to = 1 << 30;
  if (a.budget > 0) {
    const Line line = line_of(a, lane0);
    if (blockIdx.x == 0 && wave == 0) list_parts(a, line.size, lane0);
    from = up * line.size;
    if (from >= line.total) return;
    to = min(from + line.size, line.total);
    const int2 first = find_tile(a, from, lane0);
    seq = first.x;
    start = first.y;
  }
  for (;; ++seq) {
    // What depends on the lane and the sizes alone would be kept from one sequence to the next, in more registers than
    // there are; it is worked out again.
    int lane = lane0, gq = gq0, dh = a.dh;
    asm volatile("" : "+v"(lane), "+s"(gq), "+s"(dh));
    const int j = lane & 15, g = lane >> 4;
    const uint32_t model = fdiv(seq, a.by_b), b = seq - model * a.by_b.d;
    // What every load here depends on is the sequence alone, so that one wait serves them all: its length, the table's
    // entries for the wave's first two tiles, and q.
    const int begin = a.first ? max(a.first[seq], 0) : 0, length = a.lengths[seq], base = begin & ~(kTile - 1);
    const int tile_lo = max(from - start, 0);
    // The table's entry for token `lane % 32` of a tile, two tiles ahead of its use; nothing looks at it (and so waits for
    // it) before row_of, the pool's row of that token or -1 for none.
    auto look = [&](int tile) { return paged_entry(a.t, seq, static_cast<uint32_t>(base) + tile * kTile + (lane & 31)); };
    int row = look(tile_lo + wave), next = look(tile_lo + wave + NW);
    // N values of q from column d, loaded from column 0 instead of not at all, without branches that every load would
    // wait in
    const QT* q = reinterpret_cast<const QT*>(a.q) + model * a.qn + b * a.qb + (head0 + min(j, gq - 1)) * a.qh;
    constexpr int N = kF32 ? 4 : 8, NX = kF32 ? NCK : NF;
    auto column = [&](int i) {                                    // the same columns of each product as K's
      return kF32 ? (i * 4 + g) * 4 : kQ8 ? ((i / 2) * 4 + g) * 16 + (i % 2) * 8 : (i * 4 + g) * 8;
    };
    constexpr int NV = 16 / sizeof(QT);
    u32x4 raw[NX][N / NV];
#pragma unroll
    for (int i = 0; i < NX * N / NV; ++i) {
      const int d = column(i / (N / NV)) + i % (N / NV) * NV;
      u32x4& r = raw[i / (N / NV)][i % (N / NV)];
      if (a.qvec) {
        r = *reinterpret_cast<const u32x4*>(q + (d < dh ? d : 0));
      } else {
        QT v[NV];
#pragma unroll
        for (int e = 0; e < NV; ++e) v[e] = q[d + e < dh ? d + e : 0];
        __builtin_memcpy(&r, v, sizeof v);
      }
    }
    const PagedSpan span = paged_span(begin, length, a.most);
    const int seq_lo = span.lo, hi = span.hi, tiles = paged_tiles(span), tile_hi = min(tiles, to - start);
    if (a.budget == 0 && span.cut && threadIdx.x == 0) paged_fault(a.t);
    start += tiles;
    if (a.budget > 0 && tile_lo >= tile_hi) continue;             // a sequence without tokens

    u32x4 qf[kF32 ? 1 : NF][NQ];
    float q32[kF32 ? NCK : 1][4];
    f32x4 acc[NCV][CE] = {};
    float m = -INFINITY, l = 0.f;
    bool any = false;

    auto row_of = [&](int tile, int page) {
      const int tok = base + tile * kTile + (lane & 31);
      if (tile >= tile_hi || tok < seq_lo || tok >= hi) return -1;
      const int r = paged_row(a.t, page, tok, kvh);
      if (r < 0) paged_fault(a.t);
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
      for (int i = 0; i < NX; ++i) {
        QT v[N];
        float x[N];
        __builtin_memcpy(v, raw[i], sizeof v);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = j < gq && column(i) + e < dh ? to_f32(v[e]) : 0.f;
        if constexpr (kF32) {
#pragma unroll
          for (int e = 0; e < 4; ++e) q32[i][e] = x[e];
        } else {
          planes<MT, NQ>(x, qf[i]);
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
      }
      // behind the last tile too (as row 0): were there a way round these loads, the wait for V would have to be one for
      // everything in flight
      row = row_of(tile + NW, next);
      load_k(row);
      next = look(tile + 2 * NW);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
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
        p[u] = __builtin_amdgcn_exp2f(p[u] - use);
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
        if constexpr (std::is_same<QT, float>::value)
          planes<MT, NP>(p, pf);
        else
          weight_planes<MT, NP>(p, pf);
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
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // join the waves: [NW][gq][DC] outputs, then [NW][gq] maxima and sums (a sum of -1: no tokens), which become the
    // weights of the waves' outputs and, for each head, the maximum and the sum of them all
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
    if (static_cast<int>(threadIdx.x) < gq) {
      const int h = threadIdx.x;
      float mw[NW], lw[NW], top = -INFINITY, sum = 0.f;
      bool some = false;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        mw[w] = om[w * gq + h];
        lw[w] = ol[w * gq + h];
        top = fmaxf(top, mw[w]);
        some |= !(lw[w] < 0.f);
      }
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = weight2(mw[w], finite_top(top));            // 0 for a wave without tokens
        om[w * gq + h] = f;
        sum += lw[w] < 0.f ? 0.f : f * lw[w];
      }
      ol[h] = sum;
      ol[gq + h] = some;
      if (a.budget > 0) a.ml[static_cast<int64_t>(up + seq) * a.heads + head0 + h] = make_float2(top, some ? sum : -1.f);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < gq * DC / 4; i += NW * 64) {
      const int h = i / (DC / 4), d = i % (DC / 4) * 4;
      f32x4 o = {};
#pragma unroll
      for (int w = 0; w < NW; ++w) o += om[w * gq + h] * *reinterpret_cast<const f32x4*>(lds + (w * gq + h) * DC + d);
      if (a.budget == 0) {
        QT* y = reinterpret_cast<QT*>(a.o) + (static_cast<int64_t>(seq) * a.heads + head0 + h) * dh;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < dh) y[d + e] = from_f32<QT>(ol[gq + h] != 0.f ? o[e] / ol[h] : 0.f);
      } else {
        float* y = a.part + (static_cast<int64_t>(up + seq) * a.heads + head0 + h) * dh;
        if (dh % 4 == 0) {
          if (d < dh) *reinterpret_cast<f32x4*>(y + d) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < dh) y[d + e] = o[e];
        }
      }
    }
    if (a.budget == 0 || start >= to) return;
    __syncthreads();
  }
}

// Joins the parts of one (sequence, query head): their weights first, one thread a part, then their outputs, four
// columns a thread and as many parts at a time as threads remain.  It is all waiting, so a thread's first outputs are on
// their way while the weights are worked out (attention of one sequence of 4000 tokens, both kernels: 13.6 us without,
// 12.8).  VEC: rows are whole vectors.
constexpr int kAhead = 2;          // outputs that are (one 12.9, four 12.8, eight 13.0)
template <typename QT, bool VEC>
__global__ __launch_bounds__(256) void paged_join_kernel(Paged a) {
  __shared__ float weight[kTarget], out[4 * 256], red[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t at = blockIdx.x, seq = at / a.heads, head = at - seq * a.heads;
  const int2 mine = a.parts[seq];
  const int n = min(mine.y, kTarget);                              // at most the shares, which are at most kTarget
  const float2* ml = a.ml + mine.x * static_cast<int64_t>(a.heads) + head;
  const float* part = a.part + (mine.x * static_cast<int64_t>(a.heads) + head) * a.dh;
  const int quads = (a.dh + 3) / 4, rows = 256 / quads, q = tid % quads, r = tid / quads;
  auto output = [&](int s) {
    const float* p = part + s * static_cast<int64_t>(a.heads) * a.dh + q * 4;
    f32x4 v;
    if constexpr (VEC) {
      v = *reinterpret_cast<const f32x4*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = p[q * 4 + e < a.dh ? e : 0];
    }
    return v;
  };
  float2 x[kTarget / 256];
  float top = -INFINITY;
  bool some = false;
#pragma unroll
  for (int i = 0; i < kTarget / 256; ++i) {
    const int s = tid + i * 256;
    x[i] = s < n ? ml[s * static_cast<int64_t>(a.heads)] : make_float2(-INFINITY, -1.f);
    top = fmaxf(top, x[i].x);
    some |= !(x[i].y < 0.f);
  }
  f32x4 ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) ahead[i] = output(max(min(r + i * rows, n - 1), 0));
#pragma unroll
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if (lane == 0) red[wave] = top;
  some = __syncthreads_or(some);
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kTarget / 256; ++i) {
    const float f = x[i].y < 0.f ? 0.f : weight2(x[i].x, finite_top(top));
    if (tid + i * 256 < n) weight[tid + i * 256] = f;
    sum += x[i].y < 0.f ? 0.f : f * x[i].y;
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (lane == 0) red[4 + wave] = sum;
  __syncthreads();
  sum = red[4] + red[5] + red[6] + red[7];
  f32x4 o = {};
  if (r < rows) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (r + i * rows < n) o += weight[r + i * rows] * ahead[i];
#pragma unroll 4
    for (int s = r + kAhead * rows; s < n; s += rows) o += weight[s] * output(s);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e * 256 + tid] = o[e];
  __syncthreads();
  if (tid >= a.dh) return;
  float v = 0.f;
  for (int i = 0; i < rows; ++i) v += out[(tid & 3) * 256 + i * quads + tid / 4];
  reinterpret_cast<QT*>(a.o)[at * a.dh + tid] = from_f32<QT>(some ? v / sum : 0.f);
}

// Whether whole sequences may have 8 waves: over codes, whose instructions two waves a SIMD share, and where both find
// registers.  8 sequences of 600 and 1024 tokens of 2 heads of 128 columns: in 8 bits 9.8 and 13.1 us with 8 waves, 11.3
// and 15.7 with 4; in bf16 10.2 and 14.2 with 8, 9.9 and 13.5 with 4.
template <typename KT, int DC>
constexpr bool kEight = std::is_same<KT, int8_t>::value && DC <= 128;

// How the work is spread: waves in a workgroup, and the shares of the line of all tiles (0: whole sequences).
struct Plan {
  int waves, budget;
  int64_t parts;             // at most
};
Plan plan_of(const wc_paged_attn_args& p) {
  const int64_t seqs = p.cache.n * p.cache.b, heads = p.cache.heads * cdiv(p.q_heads / p.cache.heads, 16);
  const int64_t most = paged_most(p.cache, p.max_length);
  // shares for every compute unit to have as many workgroups as its registers hold, and no more: 64 sequences of
  // 1000-4000 tokens in 8 bits (three fit) took 100 us in one share a unit, 91 in two, 86 in three, 101 in four
  const int wide = p.cache.head_dim <= 64 ? 0 : p.cache.head_dim <= 128 ? 1 : 2;
  static const int kFit[2][3][3] = {{{2, 1, 1}, {3, 2, 1}, {3, 2, 1}}, {{3, 2, 1}, {4, 3, 2}, {4, 2, 1}}};
  const int target = 256 * kFit[p.cache.bits == 8][p.cache.dtype == WC_F32 ? 0 : p.cache.dtype == WC_BF16 ? 1 : 2][wide];
  // Sequences stay whole where they fill the machine by themselves, or are so short that the second launch costs more
  // than it saves: 8 sequences of 2 heads of 64 took 10.6 us whole at 1024 tokens and 14.0 in parts at 1500; of 128
  // fp32 columns 20.1 whole and 23.2 in parts at 600, 28.1 and 23.9 at 1024
  const int64_t whole = p.cache.bits == 0 && p.cache.dtype == WC_F32 && wide > 0 ? 512 : 1024;
  if (seqs * heads >= 2048 || most <= whole || !paged_countable(seqs, most))
    return Plan{seqs * heads >= 512 ? 4 : 8, 0, 0};      // 8 only where two workgroups a unit don't come anyway
  const int64_t budget = cdiv(target, heads);
  return Plan{4, static_cast<int>(budget), budget + seqs};
}
int64_t workspace_of(const wc_paged_attn_args& p, const Plan& plan) {
  if (plan.budget == 0) return 0;
  return plan.parts * p.q_heads * (((p.cache.head_dim + 1) & ~1ll) + 2) * 4 + p.cache.n * p.cache.b * 8;   // pairs stay aligned
}

template <typename QT, typename KT, int DC, int NW>
void launch(const Paged& a, int64_t grid, hipStream_t s) {
  const int gq = std::min(a.group, 16);
  const size_t lds = static_cast<size_t>(NW) * gq * (DC + 2) * sizeof(float);
  const auto kernel = paged_attention_kernel<QT, KT, DC, NW>;
  if (lds > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
  kernel<<<static_cast<uint32_t>(grid), NW * 64, lds, s>>>(a);
}

template <typename QT>
void dispatch(const Paged& a, bool q8, int waves, int64_t grid, hipStream_t s) {
  auto go = [&](auto k, auto dc) {
    typedef decltype(k) KT;
    constexpr int DC = decltype(dc)::value;
    if constexpr (kEight<KT, DC>)
      if (waves == 8) return launch<QT, KT, DC, 8>(a, grid, s);
    launch<QT, KT, DC, 4>(a, grid, s);
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
  return workspace_of(*args, plan_of(*args));
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
  a.t = paged_table(c, p.lengths);
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
  a.seqs = static_cast<int32_t>(seqs);
  a.heads = static_cast<int32_t>(p.q_heads);
  a.group = static_cast<int32_t>(p.q_heads / c.heads);
  const int64_t qtiles = cdiv(a.group, 16);
  a.dh = static_cast<int32_t>(c.head_dim);
  a.row_bytes = static_cast<int32_t>(c.row * paged_es(c));
  // the bound of plan_of's count too; a pool without pages has no row 0, a table without entries no tokens
  a.most = static_cast<int32_t>(paged_most(c, p.max_length));
  a.scale = p.scale * kLog2e;
  a.qvec = c.head_dim * es % 16 == 0 && aligned(p.q, 16) && ubytes(p.q_stride_n, es) % 16 == 0 &&
           ubytes(p.q_stride_b, es) % 16 == 0 && ubytes(p.q_stride_h, es) % 16 == 0;
  const Plan plan = plan_of(p);
  const int64_t need = workspace_of(p, plan);
  WC_REQUIRE(need == 0 || (p.workspace && p.workspace_bytes >= need), WC_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what,
             (long long)p.workspace_bytes, (long long)need);
  WC_REQUIRE(need == 0 || aligned(p.workspace, 16), WC_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  a.budget = plan.budget;
  a.part = nullptr;
  a.ml = nullptr;
  a.parts = nullptr;
  if (need) {
    a.part = static_cast<float*>(p.workspace);
    a.ml = reinterpret_cast<float2*>(a.part + plan.parts * p.q_heads * ((c.head_dim + 1) & ~1ll));
    a.parts = reinterpret_cast<int2*>(a.ml + plan.parts * p.q_heads);
  }
  a.by_qtile = make_fastdiv(static_cast<uint32_t>(qtiles));
  a.by_kvh = make_fastdiv(static_cast<uint32_t>(c.heads));
  a.by_b = make_fastdiv(static_cast<uint32_t>(c.b));
  const int64_t grid = (plan.budget ? plan.budget : seqs) * c.heads * qtiles;
  const hipStream_t s = as_stream(stream);
  auto go = [&](auto t) {
    typedef decltype(t) QT;
    dispatch<QT>(a, c.bits == 8, plan.waves, grid, s);
    if (plan.budget)
      (c.head_dim % 4 ? paged_join_kernel<QT, false> : paged_join_kernel<QT, true>)<<<static_cast<uint32_t>(seqs * p.q_heads), 256, 0, s>>>(a);
  };
  if (c.dtype == WC_F32)
    go(float());
  else if (c.dtype == WC_BF16)
    go(bf16());
  else
    go(f16());
  return check_launch(what);
}
