// Internal interface of attention over shared prefixes: stretches of tokens and the sequences that read them.
#pragma once

#include "wc_answer_abi.h"
#include "wc_paged_attn.h"

namespace wc {

constexpr int kSharedTarget = 1024;  // shares of a line at most
constexpr int kSharedWaves = 4;

// Stretches of tokens and the sequences that read them
struct SharedWalk {
  PagedTable t;
  const int32_t* lengths;            // [units]
  float* part;                       // [parts][share][heads][dh]
  float2* ml;                        // [parts][share][heads]: maximum and sum, -1 where there are no tokens
  int2* parts;                       // [units]: first part and how many, where the line of all tiles is cut (budget > 0)
  int32_t units, share, budget, least, most, rows;   // least: tiles of a share at least; rows: query heads of a unit that read one key head
  FastDiv by_tiles, by_units;        // tiles of rows; units of a model
};
struct SharedAttn {
  SharedWalk walk[2];                      // prefixes, own tokens
  const char *k, *v, *q;
  const float *ks, *vs;
  char* o;
  int64_t qn, qb, qh;
  int32_t heads, group, dh, row_bytes, qvec, blocks;  // blocks: workgroups of the prefixes' walk
  FastDiv by_kvh, by_group, by_heads, by_share;
  float scale;                       // of the scores, times log2 e
};

__device__ __forceinline__ PagedSpan shared_span(const SharedWalk& w, int unit) { return paged_span(0, w.lengths[unit], w.most); }

// Where stretches are cut, the tiles of all of them count as one line, of which every workgroup (of a key head and a tile of rows)
// has an equal share however uneven the lengths are: share w is tiles [w size, (w + 1) size), of one unit or the ends and
// wholes of several.  What share w has of unit s is part w + s: no two are alike, a unit's parts are neighbours, and there
// are at most shares + units of them.  Every wave finds its share from the lengths by itself.
struct SharedLine {
  int size, total;
};
// Tiles of a share, one at least, where there are none at all too: units' first shares are counted by dividing by it.  `least` is for
// cuts of one unit: short units are not put together for it, which would walk them one after the other.
__host__ __device__ inline int shared_size(int total, int budget, int least, int units) {
  const int equal = (total + budget - 1) / budget, low = (total + units - 1) / (units > 1 ? units : 1);
  const int size = least < low ? least : low;
  return size > equal ? size : equal > 1 ? equal : 1;
}
__device__ __forceinline__ SharedLine shared_line(const SharedWalk& w, int lane) {
  int total = 0;
  for (int s = lane; s < w.units; s += 64) total += paged_tiles(shared_span(w, s));
#pragma unroll
  for (int off = 32; off; off >>= 1) total += __shfl_xor(total, off, 64);
  return SharedLine{shared_size(total, w.budget, w.least, w.units), total};
}
// the unit that has tile `at` of the line (at < total), and the line's tiles before it
__device__ __forceinline__ int2 shared_find(const SharedWalk& w, int at, int lane) {
  int done = 0;
  for (int s0 = 0; s0 < w.units; s0 += 64) {
    const int s = s0 + lane, n = s < w.units ? paged_tiles(shared_span(w, s)) : 0;
    const int start = done + before(n, lane);
    const uint64_t mine = __ballot(at >= start && at < start + n);
    if (mine) {
      const int l = __ffsll(static_cast<unsigned long long>(mine)) - 1;
      return make_int2(s0 + l, __shfl(start, l, 64));
    }
    done = __shfl(start + n, 63, 64);
  }
  return make_int2(w.units, 0);
}
// each unit's first part and how many it has, for the kernel that joins them; and the fault of lengths that were cut
__device__ __forceinline__ void shared_list(const SharedWalk& w, int size, int lane) {
  int done = 0;
  for (int s0 = 0; s0 < w.units; s0 += 64) {
    const int s = s0 + lane;
    const PagedSpan span = s < w.units ? shared_span(w, s) : PagedSpan{0, 0, false};
    if (span.cut) paged_fault(w.t);
    const int n = paged_tiles(span);
    const int start = done + before(n, lane), w0 = start / size;
    if (s < w.units) w.parts[s] = n ? make_int2(w0 + s, (start + n - 1) / size - w0 + 1) : make_int2(0, 0);
    done = __shfl(start + n, 63, 64);
  }
}


// The prefixes' walk through LDS (shared_stream.hip), for more than 32 rows in 16 bits of head dims up to 128: rows that a
// workgroup has, 64 or 128, or 0 where it does not take the call.
int shared_stream_rows(const wc_shared_attn_args& p);
void shared_stream(const SharedAttn& a, int32_t dtype, bool q8, int rows, int64_t grid, hipStream_t s);

}  // namespace wc
