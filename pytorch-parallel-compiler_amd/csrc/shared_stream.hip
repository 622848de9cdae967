// The walk of shared prefixes through LDS: for more than 32 rows (query heads of all sequences of a prefix) to a key head, in
// 16 bits, over pages in the queries' type or of 8-bit codes.
//
// A workgroup of four waves has 128 rows, 32 a wave (or 64, of which two waves have the same and half of the tokens each),
// and walks its share of a prefix in tiles of 64 tokens, K and V row-major in LDS, double-buffered: 16-bit pages come by LDS-DMA
// issued one tile ahead, 8-bit ones through registers, as 16-bit numbers that hold the codes exactly.  Which rows of
// the pool a tile has, the lanes find from 64 entries of the table, which they hold.  Per tile and wave, with v_mfma_f32_32x32x16:
//   S^T = K Q^T      lane l holds row l % 32 and tokens 8 (r / 4) + 4 (l / 32) + r % 4 of each block of 32
//   softmax          in the lane; the lane halves that share a row exchange their maxima, and O is rescaled, only in tiles where
//                    a lane of the wave finds a score well over the row's base
//   O^T += V^T P^T   P^T is the S^T register block itself, V^T through ds_read_b64_tr_b16
// A row's K scale multiplies its scores, its V scale its weights.  The weights enter the products as two numbers of 16 bits each, off by at
// most 2^-16 of a weight (bf16; fp16 2^-21), so that a row's result does not hang on how many others share its prefix; over 8-bit
// pages as bf16 ones, because fp16 has no room for a weight times a scale.  Their sum is fp32.
//
// 64 rows are bound by memory and the waits for each tile: 4 x 2 prefixes of up to 6000 tokens, 8 key heads of 128 columns, 147 MB in
// 42 us (3.5 TB/s; four buffers and one workgroup a unit 49).  128 rows are
// bound by the matrix and vector pipes in turn: one prefix of 65536 tokens, 256 rows a key head, 132 us for 1.03e11 operations,
// which a large product does in 82 (weights rounded to 16 bits once: 105 us for 6.9e10; the 64 rows above take 42 us either way).
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

// The fragments of V^T of 16 tokens by 32 columns each, at LDS byte addresses `at` + OFF and, 8 tokens on, OFF + NEXT.  Written as
// one block with its wait, because the compiler has the builtin wait for all loads into LDS that are on their way.
template <int OFF, int NEXT>
__device__ __forceinline__ void read_v(const uint32_t (&at)[2], i16x4 (&v)[2][2]) {
  asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
               "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1])
               : "v"(at[0]), "v"(at[1]), "n"(OFF), "n"(OFF + NEXT) : "memory");
}
template <int OFF, int NEXT>
__device__ __forceinline__ void read_v(const uint32_t (&at)[4], i16x4 (&v)[4][2]) {
  asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
               "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
               "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
               "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[3][0]),
                 "=&v"(v[3][1])
               : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(OFF), "n"(OFF + NEXT) : "memory");
}

// T: type of q and o; KT: stored type; DHP: columns provided for; RW: waves that have rows of their own
template <typename T, typename KT, int DHP, int RW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void shared_stream_kernel(SharedAttn a) {
  constexpr bool kQ8 = std::is_same<KT, int8_t>::value;
  typedef typename std::conditional<kQ8, bf16, T>::type PT;            // of P and V
  constexpr int NP = 2;                                                // numbers of a weight
  // fp16 weights are taken 2^14 times as large, so that those far under 1 keep their bits (and as the other walk takes them)
  constexpr float kShift = std::is_same<PT, f16>::value ? 14.f : 0.f;
  // A row's base stays while its scores are no more than this above it: weights are then up to 2^8 (fp16: 2^15 with their shift), and
  // most tiles rescale nothing.
  constexpr float kOver = std::is_same<PT, f16>::value ? 1.f : 8.f;
  constexpr int NKS = DHP / 16, DT = DHP / 32, TILE = kStBK * DHP;
  constexpr int TS = 4 / RW, NB = 2 / TS;            // waves that share rows; blocks of 32 tokens of a wave
  constexpr int CPR = DHP * static_cast<int>(sizeof(KT)) / 16, CH = kStBK * CPR, PIECES = 2 * CH / 256;     // 16-byte pieces of a row, of a tile; a thread's
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][2 * TILE];           // [buffer][K tile, V tile]
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
  // This thread's pieces of a tile, those of K first: their rows are a whole number of swizzles apart, so that all of K have the same
  // column (16 bits: that which goes to the piece's place; 8 bits: that which is brought), and all of V.
  constexpr int kPer = CH / 256, kApart = 256 / CPR;
  static_assert(CH % 256 == 0 && kApart % 16 == 0, "pieces of a thread are whole swizzles apart");
  const int prow = tid / CPR;
  const int kcol = kQ8 ? tid % CPR * 16 : k_at<DHP>(prow, tid % CPR) - prow * DHP;
  const int vcol = kQ8 ? kcol : v_at<DHP>(prow, tid % CPR * 8) - prow * DHP;
  const bool kin = kcol * static_cast<int>(sizeof(KT)) < a.row_bytes, vin = vcol * static_cast<int>(sizeof(KT)) < a.row_bytes;
  const char* kp = a.k + kcol * static_cast<int>(sizeof(KT));
  const char* vp = a.v + vcol * static_cast<int>(sizeof(KT));
  uint32_t vat[DT];                                    // of the lane's V^T fragments in a tile, in bytes
#pragma unroll
  for (int d = 0; d < DT; ++d) vat[d] = v_at<DHP>(4 * hf + ((lane & 15) >> 2), 32 * d + (lane & 16) + 4 * (lane & 3)) * 2;
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
    // the same for all lanes, which the compiler is told, so that what hangs on it is branches
    const int begin = __builtin_amdgcn_readfirstlane(tile_lo * kPagedTile);
    const int end = __builtin_amdgcn_readfirstlane(min(span.hi, tile_hi * kPagedTile)), n = (end - begin + kStBK - 1) / kStBK;

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

    // The table's entries from block `held` on, one a lane: 64 blocks, which last for a page's length of tiles.  They have come
    // before anything else is brought, so that no tile waits for what is on its way behind it.
    int entries = 0, held = -64;
    // the pool's row of token `lane` of tile i, -1 for none
    auto row_of = [&](int i) __attribute__((always_inline)) {
      const int tok = begin + i * kStBK + lane;
      const int block = fdiv(tok, w.t.by_page), lo = __builtin_amdgcn_readfirstlane(block);
      if (__builtin_amdgcn_readlane(block, 63) - held >= 64) {
        held = lo;
        entries = paged_entry(w.t, unit, static_cast<uint32_t>(held + lane) * w.t.by_page.d);
        asm volatile("" : "+v"(entries));
      }
      const int page = __shfl(entries, block - held, 64);
      if (tok >= end) return -1;
      const int r = paged_row(w.t, page, tok, kvh);
      if (r < 0) paged_fault(w.t);
      return r;
    };
    u32x4 raw[kQ8 ? PIECES : 1];
    float ks = 0.f, vs = 0.f;
    // tile rows `row` (by lane) on their way into buffer `buf`; where there are none, row 0 of the pool, so that every tile is as many
    // loads of the wave
    auto fetch = [&](int buf, int row) {
      if constexpr (kQ8) {
        ks = row >= 0 ? a.ks[row] : 0.f;
        vs = row >= 0 ? a.vs[row] : 0.f;
      }
      int r[kPer];
#pragma unroll
      for (int u = 0; u < kPer; ++u) r[u] = __shfl(row, prow + u * kApart, 64);
      auto bring = [&](const char* p, bool in, int first) __attribute__((always_inline)) {
        if constexpr (kQ8) {
#pragma unroll
          for (int u = 0; u < kPer; ++u) {
            raw[first + u] = u32x4{0, 0, 0, 0};
            if (in && r[u] >= 0) raw[first + u] = *reinterpret_cast<const u32x4*>(p + static_cast<int64_t>(r[u]) * a.row_bytes);
          }
        } else if (in) {
#pragma unroll
          for (int u = 0; u < kPer; ++u)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const void*>(p + static_cast<int64_t>(max(r[u], 0)) * a.row_bytes),
                                             (__attribute__((address_space(3))) void*)(&lds[buf][(wave * 64 + (first + u) * 256) * 8]), 16, 0,
                                             0);
        }
      };
      bring(kp, kin, 0);
      bring(vp, vin, kPer);
    };
    // Rows of a tile that has come of which there are none, as zeros: their scores are taken out, but 0 times what stands there
    // may not be 0.
    auto blank = [&](int buf, uint64_t valid) {
#pragma unroll
      for (int u = 0; u < PIECES; ++u)
        if (!(valid >> (prow + u % kPer * kApart) & 1)) *reinterpret_cast<uint4*>(&lds[buf][(tid + u * 256) * 8]) = make_uint4(0, 0, 0, 0);
    };
    // 8 bits: the codes that have come, as numbers into LDS
    auto put = [&](int buf) {
      if constexpr (kQ8) {
        if (wave == 0) scales[buf][0][lane] = ks;
        if (wave == 1) scales[buf][1][lane] = vs;
#pragma unroll
        for (int u = 0; u < PIECES; ++u) {
          const bool isv = u >= kPer;
          if (!kin) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t v = raw[u][h * 2 + e / 2];
              const float f0 = byte_f32(v, (e & 1) * 2), f1 = byte_f32(v, (e & 1) * 2 + 1);
              x[e] = isv ? pack2<PT>(f0, f1) : pack2<T>(f0, f1);
            }
            const int at = isv ? TILE + v_at<DHP>(prow + (u - kPer) * kApart, kcol + h * 8) : k_at<DHP>(prow + u * kApart, kcol / 8 + h);
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

    __syncthreads();                                   // the buffers are free
    if (clear_columns) {
      for (int e = tid; e < 2 * 2 * TILE / 8; e += 256) reinterpret_cast<uint4*>(&lds[0][0])[e] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      clear_columns = TS == 2;                         // where the waves' outputs meet in the buffers, again
    }
    int row = row_of(0);
    uint64_t valid = __ballot(row >= 0), coming = 0;   // which of the tokens of the tile at work and of the next there are
    fetch(0, row);
    put(0);
    for (int i = 0; i < n; ++i) {
      const int buf = i & 1;
      // the tile has come for this wave, then for all, and nobody is at the one before
      __builtin_amdgcn_s_waitcnt(0x0070);              // vmcnt(0), lgkmcnt(0)
      __syncthreads();
      if (!kQ8 && valid != ~0ull) {
        blank(buf, valid);
        __syncthreads();
      }
      const uint16_t* ks_ = lds[buf];
      const uint32_t vbase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_i16x4*)(ks_ + TILE)));
      if (i + 1 < n) {
        row = row_of(i + 1);
        coming = __ballot(row >= 0);
        fetch(buf ^ 1, row);
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
            const f32x4 f = *reinterpret_cast<const f32x4*>(&scales[buf][0][32 * blk + q * 8 + 4 * hf]);
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
      if (__builtin_amdgcn_ballot_w64(fresh || bm > base + kOver) != 0) {
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
        // tokens 32 blk + 16 j + 8 piece + 4 hf + (0 .. 3), columns 32 d + 16 (lane / 16 % 2) + (0 .. 15)
        uint32_t at[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) at[d] = vbase + vat[d] + (TS == 1 ? 0 : tw * NB * 32 * DHP * 2);
        float l0 = 0.f, l1 = 0.f;
        auto half = [&](auto J) __attribute__((always_inline)) {
          constexpr int j = decltype(J)::value;
          float p[8];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * j + 2 * r], c, kShift - base));
            float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * j + 2 * r + 1], c, kShift - base));
            l0 += p0;
            l1 += p1;
            if constexpr (kQ8) {
              const float* f = &scales[buf][1][32 * blk + (2 * j + (r >> 1)) * 8 + 4 * hf + (r & 1) * 2];
              p0 *= f[0];
              p1 *= f[1];
            }
            p[2 * r] = p0;
            p[2 * r + 1] = p1;
          }
          u32x4 pf[NP];
          weight_planes<PT, NP>(p, pf);
          i16x4 v[DT][2];
          if (b == 0) read_v<j * 16 * DHP * 2, 8 * DHP * 2>(at, v);
          else read_v<(32 + j * 16) * DHP * 2, 8 * DHP * 2>(at, v);
#pragma unroll
          for (int q = NP - 1; q >= 0; --q)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const i16x8 vf = __builtin_shufflevector(v[d][0], v[d][1], 0, 1, 2, 3, 4, 5, 6, 7);
              oacc[d] = mma32<PT>(__builtin_bit_cast(bf16x8, vf), __builtin_bit_cast(bf16x8, pf[q]), oacc[d]);
            }
        };
        half(std::integral_constant<int, 0>());
        half(std::integral_constant<int, 1>());
        lrun += l0 + l1;
      }
      if (i + 1 < n) put(buf ^ 1);
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

// Up to 32 rows the walk without LDS reads a prefix once as well and needs no barriers; from there on it reads it again for every 32
// (64 rows: 86.0 us for the whole call of the case above, and 84.7 through LDS; 256 rows: 386 and 188).
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
