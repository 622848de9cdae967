/*
 * wc_serve_abi.h -- C ABI of the decode-step kernels of libwide_hip.so (gfx950 / MI355X):
 * ensembles of N language models that answer token by token.
 *
 * These operators have no counterpart in the reference, so they are declared apart from wc_abi.h
 * and have a version of their own.  Its conventions hold here too: device pointers, strides in
 * elements, launches on `stream`, nothing allocated, 0 / negative / positive status codes and
 * wc_last_error().
 *
 * A sequence is one of the n * b of a call; per-sequence tables are contiguous [n, b].
 */
#ifndef WC_SERVE_ABI_H
#define WC_SERVE_ABI_H

#include "wc_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define WC_SERVE_ABI_VERSION 1

/* Version of this header compiled into the library (== WC_SERVE_ABI_VERSION). */
int32_t wc_serve_abi_version(void);

/*
 * RMS norm of every query and key head, then the rotation by position:
 *   y = x / sqrt(mean(x^2) + eps) * weight[model]        over head_dim
 *   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)   for pair p < rotary_dim / 2
 * with the angle 2 pi position freq[p], taken in 64 bits.  Pair p is (2p, 2p + 1) when interleaved,
 * else (p, p + rotary_dim / 2); columns from rotary_dim on are not turned.
 */
typedef struct wc_head_norm_args {
  int32_t dtype, param_dtype;     /* of q, k and outputs; of the weights */
  int32_t interleaved;
  int32_t position_bytes;         /* 4 or 8: int32 or int64 positions */
  int64_t n, b, t;                /* models, sequences, tokens */
  int64_t q_heads, k_heads;       /* >= 0 */
  int64_t head_dim, rotary_dim;   /* even; 0 <= rotary_dim <= head_dim <= 256 */
  const void* q;                  /* [n, b, t, q_heads, head_dim], unit stride over head_dim */
  int64_t q_stride_n, q_stride_b, q_stride_t, q_stride_h;
  const void* k;                  /* [n, b, t, k_heads, head_dim] */
  int64_t k_stride_n, k_stride_b, k_stride_t, k_stride_h;
  void* q_out;                    /* contiguous [n, b, t, q_heads, head_dim] */
  void* k_out;                    /* contiguous [n, b, t, k_heads, head_dim] */
  const void* q_weight;           /* [n, head_dim] contiguous */
  const void* k_weight;
  const double* freq;             /* [rotary_dim / 2]: turns per position */
  const void* positions;          /* [n, b, t] through the strides below (0 for broadcast) */
  int64_t p_stride_n, p_stride_b, p_stride_t;
  float eps;
} wc_head_norm_args;

int32_t wc_head_norm_rotary(const wc_head_norm_args* args, void* stream);

/*
 * A paged key-value cache.  Token i of a sequence is row i % page_size of the page that entry
 * i / page_size of the sequence's block table names; K and V rows of a head stand at
 *   pages + ((page * heads + head) * page_size + slot) * row      (row elements, head_dim of them used)
 * in `dtype` (bits 0), or as 8-bit codes (bits 8) with one fp32 scale at the same index of the scales:
 *   scale = max(max |x| / 127, 2^-126),  code = x / scale to the nearest, ties to even (exactly),
 * (a unit of the last place less for the largest fp32 value, so that 127 times it is finite),
 * and a row that holds an infinity or NaN gets scale NaN and codes 0: it reads back as NaN.
 * A table entry outside [0, pages), or a token past the table's end, is never followed: its row is
 * not written, reads as zeros, takes no part in the attention, and stores 1 in *err_flag.
 */
typedef struct wc_paged_cache {
  int32_t dtype, bits;
  int64_t n, b;
  int64_t pages, page_size, heads, head_dim;    /* head_dim <= 256 */
  int64_t row;                    /* elements; whole 16-byte vectors; those past head_dim hold 0 */
  void* k_pages;
  void* v_pages;                  /* 16-byte aligned */
  float* k_scales;
  float* v_scales;                /* bits 8 only */
  const int32_t* table;           /* [n, b, table_len], row stride table_stride */
  int64_t table_len, table_stride;
  int32_t* err_flag;              /* may be NULL */
} wc_paged_cache;

/* Writes tokens [start, start + count) of every sequence from rows [0, count) of k and v; count NULL: all
 * t rows.  A sequence of negative start takes part in nothing.  No two rows of a call may go to one place of the
 * pool. */
typedef struct wc_cache_write_args {
  wc_paged_cache cache;
  int64_t t;
  const void* k;                  /* [n, b, t, heads, head_dim] of cache.dtype, unit stride over head_dim */
  int64_t k_stride_n, k_stride_b, k_stride_t, k_stride_h;
  const void* v;
  int64_t v_stride_n, v_stride_b, v_stride_t, v_stride_h;
  const int32_t* start;           /* [n, b] */
  const int32_t* count;           /* [n, b] or NULL */
} wc_cache_write_args;

int32_t wc_cache_write(const wc_cache_write_args* args, void* stream);

/* Reads tokens [0, length) of every sequence into k, v [n, b, max_length, heads, head_dim] (contiguous, of
 * cache.dtype); rows from a sequence's length on are zeros. */
typedef struct wc_cache_read_args {
  wc_paged_cache cache;
  const int32_t* lengths;         /* [n, b]; at most max_length of a sequence's tokens are read */
  int64_t max_length;
  void* k;
  void* v;
} wc_cache_read_args;

int32_t wc_cache_read(const wc_cache_read_args* args, void* stream);

/*
 * Attention of one new token of every sequence over its cached tokens [first, length):
 *   o[h] = sum_i softmax_i(scale * q[h] . k_i) v_i,   key head h / (q_heads / cache.heads)
 * A sequence without tokens gets zeros.  max_length bounds the lengths (longer ones are cut there and
 * raise the error flag) and sets how far the work is split over a sequence.
 */
typedef struct wc_paged_attn_args {
  wc_paged_cache cache;
  int64_t q_heads;                /* a multiple of cache.heads */
  int64_t max_length;
  const void* q;                  /* [n, b, q_heads, head_dim], unit stride over head_dim */
  int64_t q_stride_n, q_stride_b, q_stride_h;
  void* o;                        /* contiguous [n, b, q_heads, head_dim] */
  const int32_t* lengths;         /* [n, b] */
  const int32_t* first;           /* [n, b] or NULL (0) */
  void* workspace;                /* wc_paged_attention_workspace_bytes(args), 16-byte aligned */
  int64_t workspace_bytes;
  float scale;
} wc_paged_attn_args;

/* Bytes of workspace (0: none is needed), or -1 for sizes that wc_paged_attention rejects. */
int64_t wc_paged_attention_workspace_bytes(const wc_paged_attn_args* args);

int32_t wc_paged_attention(const wc_paged_attn_args* args, void* stream);

/*
 * y = x W^T + bias with W of 4-bit codes: W[o, k] = scale[o, k / group] (code[o, k] - zero[o, k / group]).
 * The weights are stored in tiles of 16 rows x 128 columns (rows and columns padded with code 0, groups
 * with scale 0):
 *   codes   [n, row tiles, column tiles, 64, 4] 32-bit words; word q of lane l holds row l % 16 and columns
 *           32 q + 8 (l / 16) + e of the tile, e = 0..7 in nibbles 0, 4, 1, 5, 2, 6, 3, 7
 *   scales  [n, row tiles, column tiles * 128 / group, 16] of `dtype`
 *   zeros   the same of uint8, each at most 127
 */
typedef struct wc_linear4_args {
  int32_t dtype;                  /* of x, scales, bias and y */
  int32_t group;                  /* 32, 64 or 128 */
  int64_t n, m, o, k;
  const void* x;                  /* row r of model i at i * stride_n + (r / rows_inner) * stride_outer
                                     + (r % rows_inner) * stride_inner, unit stride over k */
  int64_t x_stride_n, x_stride_outer, x_stride_inner, x_rows_inner;
  const void* codes;
  const void* scales;
  const void* zeros;
  const void* bias;               /* [n, o] or NULL */
  void* y;                        /* contiguous [n, m, o] */
} wc_linear4_args;

int32_t wc_linear4(const wc_linear4_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* WC_SERVE_ABI_H */
