// What the kernels over a paged key-value cache share: its addressing and the host checks of its description.
#pragma once

#include <algorithm>

#include "wc_common.h"
#include "wc_serve_abi.h"

namespace wc {

struct PagedTable {
  const int32_t* table;
  int64_t stride;
  int32_t len, pages, page, heads;
  int32_t* err;
  FastDiv by_page;
};

// The table's entry for token `tok` of sequence `seq`, behind its end the last: loaded without a condition, so that
// neighbouring loads need not wait for each other
__device__ __forceinline__ int32_t paged_entry(const PagedTable& t, int64_t seq, uint32_t tok) {
  return t.table[seq * t.stride + min(fdiv(tok, t.by_page), static_cast<uint32_t>(max(t.len, 1) - 1))];
}
// The row of the pool (in units of rows) that holds token `tok` for head `h` in page `id` of the table, or -1 where the
// table has none.  Rows of a pool fit 31 bits (paged_check).
__device__ __forceinline__ int32_t paged_row(const PagedTable& t, int32_t id, uint32_t tok, int h) {
  const uint32_t block = fdiv(tok, t.by_page);
  if (block >= static_cast<uint32_t>(t.len) || static_cast<uint32_t>(id) >= static_cast<uint32_t>(t.pages)) return -1;
  return (id * t.heads + h) * t.page + static_cast<int32_t>(tok - block * t.by_page.d);
}

__device__ __forceinline__ void paged_fault(const PagedTable& t) {
  if (t.err) *t.err = 1;
}

// instead: as many int32 as there are sequences, for a table without entries, of which one is loaded all the same
inline PagedTable paged_table(const wc_paged_cache& c, const int32_t* instead) {
  PagedTable t;
  t.table = c.table_len ? c.table : instead;
  t.stride = c.table_len ? c.table_stride : 0;
  t.len = static_cast<int32_t>(c.table_len);
  t.pages = static_cast<int32_t>(c.pages);
  t.page = static_cast<int32_t>(c.page_size);
  t.heads = static_cast<int32_t>(c.heads);
  t.err = c.err_flag;
  t.by_page = make_fastdiv(static_cast<uint32_t>(c.page_size));
  return t;
}

// What attention walks: a sequence's tokens [lo, hi) in tiles of kPagedTile, counted from the one that holds token lo.
constexpr int kPagedTile = 32;
struct PagedSpan {
  int32_t lo, hi;
  bool cut;                  // the length was beyond most
};
__host__ __device__ inline PagedSpan paged_span(int32_t first, int32_t length, int32_t most) {
  return PagedSpan{first > 0 ? first : 0, length < most ? length : most, length > most};
}
__host__ __device__ inline int32_t paged_tiles(const PagedSpan& s) {
  return s.hi > s.lo ? (s.hi - (s.lo & ~(kPagedTile - 1)) + kPagedTile - 1) / kPagedTile : 0;
}
// The tokens that a sequence has at most, whatever its length says: those its table can name and max_length allows, which
// is under 2^31 - 64; none of a pool without pages.
inline int64_t paged_most(const wc_paged_cache& c, int64_t max_length) {
  return c.pages ? std::min(max_length, c.table_len * c.page_size) : 0;
}
// Whether the tiles of all sequences, and a share's end behind the last of them, can be counted in 32 bits
inline bool paged_countable(int64_t seqs, int64_t most) {
  return mul_sat({seqs, (most + kPagedTile - 1) / kPagedTile}) < (1ll << 30);
}

// Bytes of a stored element
inline int paged_es(const wc_paged_cache& c) { return c.bits == 8 ? 1 : dtype_size(c.dtype); }

// Sizes and types of a cache; its pointers are checked by paged_check_pointers once a call has work to do.
inline int32_t paged_check(const wc_paged_cache& c, const char* what) {
  WC_REQUIRE(dtype_size(c.dtype), WC_ERR_DTYPE, "%s: dtype %d", what, c.dtype);
  WC_REQUIRE(c.bits == 0 || c.bits == 8, WC_ERR_DTYPE, "%s: bits %d (0 or 8)", what, c.bits);
  WC_REQUIRE(c.n >= 0 && c.b >= 0 && c.pages >= 0 && c.heads >= 0 && c.table_len >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(c.page_size > 0 && c.head_dim > 0 && c.row >= c.head_dim, WC_ERR_SHAPE,
             "%s: page_size, head_dim and row must be positive, row at least head_dim", what);
  WC_REQUIRE(c.head_dim <= 256, WC_ERR_LIMIT, "%s: head_dim %lld above 256", what, (long long)c.head_dim);
  WC_REQUIRE(c.row <= 512 && c.row * paged_es(c) % 16 == 0, WC_ERR_ALIGN, "%s: rows of %lld elements (whole 16-byte vectors, at most 512)",
             what, (long long)c.row);
  WC_REQUIRE(mul_sat({c.n, c.b}) < (1ll << 24) && c.table_len < (1ll << 31) && mul_sat({c.pages, c.heads, c.page_size}) < (1ll << 31) &&
                 c.page_size <= (1 << 24) && c.heads <= 65535 && c.pages < (1ll << 31),
             WC_ERR_LIMIT, "%s: more than 2^24 sequences, 2^31 rows in the pool or 65535 heads, or pages above 2^24 tokens", what);
  WC_REQUIRE(c.table_len <= 1 || c.table_stride >= 0, WC_ERR_ARG, "%s: negative table stride", what);
  return WC_OK;
}

inline int32_t paged_check_pointers(const wc_paged_cache& c, const char* what) {
  // a pool without rows is never followed; neither is a table without entries
  const bool rows = c.pages > 0 && c.heads > 0;
  WC_REQUIRE((!rows || (c.k_pages && c.v_pages && (c.bits == 0 || (c.k_scales && c.v_scales)))) && (c.table_len == 0 || c.table),
             WC_ERR_NULL, "%s: null cache pointer", what);
  WC_REQUIRE(aligned(c.k_pages, 16) && aligned(c.v_pages, 16) && aligned(c.k_scales, 4) && aligned(c.v_scales, 4) &&
                 aligned(c.table, 4) && aligned(c.err_flag, 4),
             WC_ERR_ALIGN, "%s: pages must be 16-byte aligned, tables 4-byte", what);
  return WC_OK;
}

}  // namespace wc
