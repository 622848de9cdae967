// The walk of shared prefixes through LDS: for more than 32 rows (query heads of all sequences of a prefix) to a key head, in
// 16 bits, over pages in the queries' type or of 8-bit codes.
//
// A workgroup of four waves has 128 rows, 32 a wave (or 64, of which two waves have the same and half of the tokens each),
// and walks its share of a prefix in tiles of 64 tokens, K and V row-major in LDS, double-buffered: 16-bit pages come by LDS-DMA
// issued one tile ahead, 8-bit ones through registers, as 16-bit numbers that hold the codes exactly.  Which rows of
// the pool a tile has, the lanes find from the table two tiles ahead.  Per tile and wave, with v_mfma_f32_32x32x16:
//   S^T = K Q^T      lane l holds row l % 32 and tokens 8 (r / 4) + 4 (l / 32) + r % 4 of each block of 32
//   softmax          in the lane; the lane halves that share a row exchange their maxima, and O is rescaled, only in tiles where
//                    a lane of the wave finds a new running maximum
//   O^T += V^T P^T   P^T is the S^T register block itself, V^T through ds_read_b64_tr_b16
// A row's K scale multiplies its scores, its V scale its weights.  The weights enter the products rounded to 16 bits, half a step
// of 2^-8 (bf16) or 2^-11 (fp16) of each, as in attention over a prompt; their sum is fp32.  fp16 over 8-bit pages takes
// them as two bf16 numbers, because fp16 has no room for a weight times a scale.
#include "wc_attn.h"
#include "wc_shared.h"

namespace wc {
namespace {

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

template <typename T>
__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) {
  if constexpr (std::is_same<T, f16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// T: type of q and o; KT: stored type; DHP: columns provided for; RW: waves that have rows of their own
template <typename T, typename KT, int DHP, int RW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void shared_stream_kernel(SharedAttn a) {
  constexpr bool kQ8 = std::is_same<KT, int8_t>::value;
  typedef typename std::conditional<kQ8, bf16, T>::type PT;            // of P and V
  constexpr int NP = kQ8 && std::is_same<T, f16>::value ? 2 : 1;
  // fp16 weights are taken 2^14 times as large, so that those far under 1 keep their bits (and as the other walk takes them)
  constexpr float kShift = std::is_same<PT, f16>::value ? 14.f : 0.f;
  constexpr int NKS = DHP / 16, DT = DHP / 32, TILE = kStBK * DHP;
  constexpr int TS = 4 / RW, NB = 2 / TS;            // waves that share rows; blocks of 32 tokens of a wave
  constexpr int CPR = DHP * static_cast<int>(sizeof(KT)) / 16, CH = kStBK * CPR, PIECES = 2 * CH / 256;     // 16-byte pieces of a row, of a tile; a thread's
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][2 * TILE];   // [buffer][K tile, V tile]
  __shared__ float scales[kQ8 ? 2 : 1][2][kStBK];
  const SharedWalk& w = a.walk[0];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5, rw = wave % RW, tw = wave / RW;
  // neighbours, which are tiles of rows over the same tokens, on one XCD
  uint32_t id = blockIdx.x;
  if (gridDim.x % 8 == 0) id = (id & 7) * (gridDim.x >> 3) + (id >> 3);
  uint32_t up = fdiv(id, w.by_tiles);
  const int row0 = (id - up * w.by_tiles.d) * (RW * 32);
  id = up;
  up = fdiv(id, a.by_kvh);
  const int kvh = id - up * a.by_kvh.d;
  const SharedLine line = shared_line(w, lane);
  if (id == 0 && row0 == 0 && wave == 0) shared_list(w, line.size, lane);
  const int from = up * line.size;
  if (from >= line.total) return;
  const int to = min(from + line.size, line.total);
  const int2 first = shared_find(w, from, lane);
  int unit = first.x, start = first.y;
  bool clear_columns = a.row_bytes < DHP * static_cast<int>(sizeof(KT));       // those that no row has stay zero
  // this thread's pieces of a tile: row of the tile and the column that goes to its place (16 bits), or is brought (8 bits)
  int prow[PIECES], pcol[PIECES];
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    const bool isv = wave * 64 + u * 256 >= CH;        // the same for all lanes of a wave
    const int e = tid + u * 256 - (isv ? CH : 0);
    prow[u] = e / CPR;
    const int ch = e % CPR;
    pcol[u] = kQ8 ? ch * 16 : (isv ? v_at<DHP>(prow[u], ch * 8) : k_at<DHP>(prow[u], ch)) - prow[u] * DHP;
  }
  // the maximum is that of the sums, times a positive scale: the queries take the sign, or are 0
  const float c = a.scale == 0.f ? 1.f : fabsf(a.scale);
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, keep = a.scale == 0.f ? 0u : ~0u;
  const int dh = a.dh, rows = w.rows;

  for (;; ++unit) {
    const uint32_t model = fdiv(unit, w.by_units), b0 = (unit - model * w.by_units.d) * w.share;
    const int tile_lo = max(from - start, 0);
    const PagedSpan span = shared_span(w, unit);
    const int tiles = paged_tiles(span), tile_hi = min(tiles, to - start);
    start += tiles;
    if (tile_lo >= tile_hi) continue;                 // a unit without tokens
    const int begin = tile_lo * kPagedTile, end = min(span.hi, tile_hi * kPagedTile), n = (end - begin + kStBK - 1) / kStBK;

    // Q^T fragments (B operand of S^T): row l32 of the wave's, columns 16 k + 8 hf .. + 8
    bf16x8 qf[NKS];
    {
      const int r = min(row0 + rw * 32 + l32, rows - 1);
      const uint32_t s = fdiv(r, a.by_group), h = r - s * a.by_group.d;
      const T* q = reinterpret_cast<const T*>(a.q) + model * a.qn + (b0 + s) * a.qb + (kvh * a.group + h) * a.qh;
#pragma unroll
      for (int k = 0; k < NKS; ++k) {
        const int d = 16 * k + 8 * hf;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (a.qvec) {
          if (d < dh) v = *reinterpret_cast<const uint4*>(q + d);
        } else {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = d + 2 * e < dh ? __builtin_bit_cast(uint16_t, q[d + 2 * e]) : 0;
            if (d + 2 * e + 1 < dh) x[e] |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, q[d + 2 * e + 1])) << 16;
          }
          v = make_uint4(x[0], x[1], x[2], x[3]);
        }
        v = make_uint4((v.x & keep) ^ flip, (v.y & keep) ^ flip, (v.z & keep) ^ flip, (v.w & keep) ^ flip);
        qf[k] = __builtin_bit_cast(bf16x8, v);
      }
    }

    // the table's entry and then the pool's row of token `lane` of tile i, -1 for none
    auto look = [&](int i) { return paged_entry(w.t, unit, static_cast<uint32_t>(begin) + i * kStBK + lane); };
    auto row_of = [&](int i, int page) {
      const int tok = begin + i * kStBK + lane;
      if (tok >= end) return -1;
      const int r = paged_row(w.t, page, tok, kvh);
      if (r < 0) paged_fault(w.t);
      return r;
    };
    u32x4 raw[kQ8 ? PIECES : 1];
    float ks = 0.f, vs = 0.f;
    // tile rows `row` (by lane) on their way into buffer `buf`; those there are none of as zeros: their scores are taken out, but 0
    // times what is left of an earlier tile may not be 0
    auto fetch = [&](int buf, int row) {
      if constexpr (kQ8) {
        ks = row >= 0 ? a.ks[row] : 0.f;
        vs = row >= 0 ? a.vs[row] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < PIECES; ++u) {
        const bool isv = wave * 64 + u * 256 >= CH;
        const int r = __shfl(row, prow[u], 64);
        const char* p = (isv ? a.v : a.k) + static_cast<int64_t>(max(r, 0)) * a.row_bytes + pcol[u] * static_cast<int>(sizeof(KT));
        const bool in = pcol[u] * static_cast<int>(sizeof(KT)) < a.row_bytes;
        if constexpr (kQ8) {
          raw[u] = u32x4{0, 0, 0, 0};
          if (in && r >= 0) raw[u] = *reinterpret_cast<const u32x4*>(p);
        } else {
          if (in && r >= 0)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const void*>(p),
                                             (__attribute__((address_space(3))) void*)(&lds[buf][(wave * 64 + u * 256) * 8]), 16, 0, 0);
          else if (r < 0)
            *reinterpret_cast<uint4*>(&lds[buf][(tid + u * 256) * 8]) = make_uint4(0, 0, 0, 0);
        }
      }
    };
    // 8 bits: the codes that have come, as numbers into LDS
    auto put = [&](int buf) {
      if constexpr (kQ8) {
        if (wave == 0) scales[buf][0][lane] = ks;
        if (wave == 1) scales[buf][1][lane] = vs;
#pragma unroll
        for (int u = 0; u < PIECES; ++u) {
          const bool isv = wave * 64 + u * 256 >= CH;
          if (pcol[u] >= a.row_bytes) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t v = raw[u][h * 2 + e / 2];
              const float f0 = byte_f32(v, (e & 1) * 2), f1 = byte_f32(v, (e & 1) * 2 + 1);
              x[e] = isv ? pack2<PT>(f0, f1) : pack2<T>(f0, f1);
            }
            const int at = isv ? TILE + v_at<DHP>(prow[u], pcol[u] + h * 8) : k_at<DHP>(prow[u], pcol[u] / 8 + h);
            *reinterpret_cast<u32x4*>(&lds[buf][at]) = x;
          }
        }
      }
    };

    f32x16 oacc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[d][e] = 0.f;
    // base: subtracted from the scaled scores, 0 until the row has met a score above -infinity (fresh; its sums are zero until
    // then); lrun: this lane half's part of the row's sum
    float base = 0.f, lrun = 0.f;
    bool fresh = true, any = false;

    int row = row_of(0, look(0)), next = look(1);
    __syncthreads();                                   // the buffers are free
    if (clear_columns) {
      for (int e = tid; e < 2 * 2 * TILE / 8; e += 256) reinterpret_cast<uint4*>(&lds[0][0])[e] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      clear_columns = TS == 2;                         // where the waves' outputs meet in the buffers, again
    }
    fetch(0, row);
    uint64_t valid = __ballot(row >= 0);
    put(0);
    __builtin_amdgcn_s_waitcnt(0x0070);                // vmcnt(0) lgkmcnt(0)
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      const uint16_t* ks_ = lds[i & 1];
      const uint16_t* vs_ = ks_ + TILE;
      uint64_t coming = 0;
      if (i + 1 < n) {                                 // the other buffer was last read before the previous barrier
        row = row_of(i + 1, next);
        coming = __ballot(row >= 0);
        fetch((i + 1) & 1, row);
        next = look(i + 2);
      }
      any |= valid != 0;
      f32x16 s[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int blk = TS == 1 ? b : tw * NB + b;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[b][e] = 0.f;
#pragma unroll
        for (int k = 0; k < NKS; ++k) {
          const bf16x8 kf = *reinterpret_cast<const bf16x8*>(ks_ + k_at<DHP>(32 * blk + l32, 2 * k + hf));
          s[b] = mma32<T>(kf, qf[k], s[b]);
        }
        if constexpr (kQ8) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 f = *reinterpret_cast<const f32x4*>(&scales[i & 1][0][32 * blk + q * 8 + 4 * hf]);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[b][q * 4 + e] *= f[e];
          }
        }
        if (valid != ~0ull) {
          const uint32_t bits = static_cast<uint32_t>(valid >> 32 * blk);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!(bits >> ((r >> 2) * 8 + 4 * hf + (r & 3)) & 1)) s[b][r] = -INFINITY;
        }
      }
      float bm = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float m0 = __builtin_fmaxf(__builtin_fmaxf(s[b][0], s[b][1]), s[b][2]);
        const float m1 = __builtin_fmaxf(__builtin_fmaxf(s[b][3], s[b][4]), s[b][5]);
        const float m2 = __builtin_fmaxf(__builtin_fmaxf(s[b][6], s[b][7]), s[b][8]);
        const float m3 = __builtin_fmaxf(__builtin_fmaxf(s[b][9], s[b][10]), s[b][11]);
        const float m4 = __builtin_fmaxf(__builtin_fmaxf(s[b][12], s[b][13]), s[b][14]);
        bm = __builtin_fmaxf(bm, __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(m0, m1), m2),
                                                 __builtin_fmaxf(__builtin_fmaxf(m3, m4), s[b][15])));
      }
      bm *= c;
      if (__builtin_amdgcn_ballot_w64(fresh || bm > base) != 0) {
        bm = __builtin_fmaxf(bm, __shfl_xor(bm, 32, 64));
        const bool higher = (fresh || bm > base) && bm > -INFINITY;
        const float nbase = higher ? bm : base;
        const float alpha = fresh ? 1.0f : __builtin_amdgcn_exp2f(base - nbase);
#pragma unroll
        for (int d = 0; d < DT; ++d) oacc[d] *= alpha;
        lrun *= alpha;
        base = nbase;
        fresh = fresh && !higher;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int blk = TS == 1 ? b : tw * NB + b;
        uint32_t pk[NP][8];
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][2 * r], c, kShift - base));
          float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][2 * r + 1], c, kShift - base));
          l0 += p0;
          l1 += p1;
          if constexpr (kQ8) {
            const float* f = &scales[i & 1][1][32 * blk + (r >> 1) * 8 + 4 * hf + (r & 1) * 2];
            p0 *= f[0];
            p1 *= f[1];
          }
          pk[0][r] = pack2<PT>(p0, p1);
          if constexpr (NP == 2) pk[1][r] = pack2<PT>(p0 - unpack_lo<PT>(pk[0][r]), p1 - unpack_hi<PT>(pk[0][r]));
        }
        lrun += l0 + l1;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          bf16x8 pf[NP];
#pragma unroll
          for (int q = 0; q < NP; ++q)
            pf[q] = __builtin_bit_cast(bf16x8, make_uint4(pk[q][4 * j], pk[q][4 * j + 1], pk[q][4 * j + 2], pk[q][4 * j + 3]));
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            // tokens 32 blk + 16 j + 8 piece + 4 hf + (0 .. 3), columns 32 d + 16 (lane / 16 % 2) + (0 .. 15)
            const int vr = 32 * blk + 16 * j + 4 * hf + ((lane & 15) >> 2), vc = 32 * d + (lane & 16) + 4 * (lane & 3);
            const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vs_ + v_at<DHP>(vr, vc)));
            const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vs_ + v_at<DHP>(vr + 8, vc)));
            const i16x8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int q = NP - 1; q >= 0; --q) oacc[d] = mma32<PT>(__builtin_bit_cast(bf16x8, vf), pf[q], oacc[d]);
          }
        }
      }
      if (i + 1 < n) {
        put((i + 1) & 1);
        __builtin_amdgcn_s_waitcnt(0x0070);
        __syncthreads();
      }
      valid = coming;
    }

    // the part: a row's maximum, sum and output (lane: row l32, columns 32 d + 8 (r / 4) + 4 hf + r % 4)
    float l = lrun + __shfl_xor(lrun, 32, 64), m = fresh ? -INFINITY : base;
    if constexpr (TS == 2) {
      // the waves of the other tokens, through LDS: [RW][DT * 16 + 2][64]
      float* x = reinterpret_cast<float*>(&lds[0][0]) + rw * (DT * 16 + 2) * 64 + lane;
      __syncthreads();
      if (tw == 1) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[(d * 16 + e) * 64] = oacc[d][e];
        x[DT * 16 * 64] = m;
        x[(DT * 16 + 1) * 64] = l;
      }
      __syncthreads();
      if (tw == 0) {
        const float m1 = x[DT * 16 * 64], l1 = x[(DT * 16 + 1) * 64], top = __builtin_fmaxf(m, m1);
        const float f0 = weight2(m, finite_top(top)), f1 = weight2(m1, finite_top(top));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) oacc[d][e] = f0 * oacc[d][e] + f1 * x[(d * 16 + e) * 64];
        l = f0 * l + f1 * l1;
        m = top;
      }
    }
    const int r = row0 + rw * 32 + l32;
    if (tw == 0 && r < rows) {
      const uint32_t s = fdiv(r, a.by_group);
      const int64_t at = (static_cast<int64_t>(up + unit) * w.share + s) * a.heads + kvh * a.group + (r - s * a.by_group.d);
      if (hf == 0) w.ml[at] = make_float2(m, any ? l : -1.f);
      float* y = w.part + at * dh;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = 32 * d + 8 * q + 4 * hf;
          if (dh % 4 == 0) {
            if (col < dh) *reinterpret_cast<f32x4*>(y + col) = f32x4{oacc[d][4 * q], oacc[d][4 * q + 1], oacc[d][4 * q + 2], oacc[d][4 * q + 3]};
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < dh) y[col + e] = oacc[d][4 * q + e];
          }
        }
    }
    if (start >= to) return;
  }
}

template <typename T, typename KT>
void launch(const SharedAttn& a, int rows, int64_t grid, hipStream_t s) {
  const uint32_t g = static_cast<uint32_t>(grid);
  if (a.dh <= 64)
    (rows == 64 ? shared_stream_kernel<T, KT, 64, 2> : shared_stream_kernel<T, KT, 64, 4>)<<<g, 256, 0, s>>>(a);
  else
    (rows == 64 ? shared_stream_kernel<T, KT, 128, 2> : shared_stream_kernel<T, KT, 128, 4>)<<<g, 256, 0, s>>>(a);
}

}  // namespace

int shared_stream_rows(const wc_shared_attn_args& p) {
  const int64_t rows = p.share * (p.q_heads / p.cache.heads);
  if (p.cache.dtype == WC_F32 || p.cache.head_dim > 128 || rows <= 32) return 0;
  return rows <= 64 ? 64 : 128;
}

void shared_stream(const SharedAttn& a, int32_t dtype, bool q8, int rows, int64_t grid, hipStream_t s) {
  if (dtype == WC_BF16)
    q8 ? launch<bf16, int8_t>(a, rows, grid, s) : launch<bf16, bf16>(a, rows, grid, s);
  else
    q8 ? launch<f16, int8_t>(a, rows, grid, s) : launch<f16, f16>(a, rows, grid, s);
}

}  // namespace wc
