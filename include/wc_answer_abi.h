/*
 * wc_answer_abi.h -- C ABI of the kernels of libwide_hip.so (gfx950 / MI355X) for ensembles of N language models that
 * draw many answers to the same prompts: attention over a prefix that sequences share, products in 8-bit integers,
 * sampling.
 *
 * These operators have no counterpart in the reference, so they are declared apart from wc_abi.h, and with a version of
 * their own apart from wc_serve_abi.h, whose conventions and paged cache they take: device pointers, strides in elements,
 * launches on `stream`, nothing allocated, 0 / negative / positive status codes and wc_last_error().
 */
#ifndef WC_ANSWER_ABI_H
#define WC_ANSWER_ABI_H

#include "wc_serve_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define WC_ANSWER_ABI_VERSION 1

/* Version of this header compiled into the library (== WC_ANSWER_ABI_VERSION). */
int32_t wc_answer_abi_version(void);

/*
 * Attention of one new token of every sequence over a prefix that `share` neighbouring sequences of a model have in common,
 * and over tokens of its own:
 *   o[h] = sum_i softmax_i(scale * q[h] . k_i) v_i,   key head h / (q_heads / cache.heads)
 * with i over tokens [0, prefix_lengths[n, b / share]) of row b / share of the model's prefix_table and tokens
 * [0, lengths[n, b]) of row b of cache.table.  A sequence of negative length takes part in nothing and gets zeros, as does
 * one without tokens.  max_prefix and max_length bound the lengths (longer ones are cut there and raise the error
 * flag) and set how far the work is split.
 */
typedef struct wc_shared_attn_args {
  wc_paged_cache cache;           /* table: the sequences' own pages, [n, b, table_len] */
  int64_t share;                  /* sequences of a prefix; divides b */
  const int32_t* prefix_table;    /* [n, b / share, prefix_len], row stride prefix_stride */
  int64_t prefix_len, prefix_stride;
  const int32_t* prefix_lengths;  /* [n, b / share] */
  int64_t q_heads;                /* a multiple of cache.heads */
  int64_t max_prefix, max_length;
  const void* q;                  /* [n, b, q_heads, head_dim], unit stride over head_dim */
  int64_t q_stride_n, q_stride_b, q_stride_h;
  void* o;                        /* contiguous [n, b, q_heads, head_dim] */
  const int32_t* lengths;         /* [n, b] */
  void* workspace;                /* wc_shared_attention_workspace_bytes(args), 16-byte aligned */
  int64_t workspace_bytes;
  float scale;
} wc_shared_attn_args;

/* Bytes of workspace, or -1 for sizes that wc_shared_attention rejects. */
int64_t wc_shared_attention_workspace_bytes(const wc_shared_attn_args* args);

int32_t wc_shared_attention(const wc_shared_attn_args* args, void* stream);

/*
 * y = x W^T + bias in 8-bit integers: each row of x becomes codes and a scale,
 *   s = max(max |x| / 127, 2^-126),  c = x / s to the nearest, ties to even (exactly),
 * and y[r, o] = s[r] scales[o] sum_k c[r, k] codes[o, k] + bias[o], the sum in 32-bit integers.  A row with an infinity or
 * NaN gives NaN.  Codes of weights stand in tiles of 16 rows x 64 columns, rows padded to a multiple of 16 and columns to
 * one of 128 with code 0:
 *   codes  [n, row tiles, column tiles, 64, 16] int8; byte e of lane l holds row l % 16 and column 16 (l / 16) + e
 */
typedef struct wc_linear8_args {
  int32_t dtype;                  /* of x, bias and y */
  int64_t n, m, o, k;             /* k at most 131072 */
  const void* x;                  /* row r of model i at i * stride_n + (r / rows_inner) * stride_outer
                                     + (r % rows_inner) * stride_inner, unit stride over k */
  int64_t x_stride_n, x_stride_outer, x_stride_inner, x_rows_inner;
  const void* codes;
  const float* scales;            /* [n, o] */
  const void* bias;               /* [n, o] or NULL */
  void* y;                        /* contiguous [n, m, o] */
  void* workspace;                /* wc_linear8_workspace_bytes(args), 16-byte aligned */
  int64_t workspace_bytes;
} wc_linear8_args;

/* Bytes of workspace, or -1 for sizes that wc_linear8 rejects. */
int64_t wc_linear8_workspace_bytes(const wc_linear8_args* args);

int32_t wc_linear8(const wc_linear8_args* args, void* stream);

/*
 * Draws a token of every row of logits from the random number u of that row:
 *   w_i = exp((x_i - max x) / temperature),  kept: the first of the order (value down, index up) such that there are at
 *   most top_k, each but the first follows less than top_p of the weight of those that top_k leaves, and w_i >= min_p;
 *   token = the lowest kept i with  sum of the kept w up to i  >  u * sum of all kept w.
 * temperature <= 0 takes the first of the order; top_k <= 0, top_p >= 1 and min_p <= 0 filter nothing, and the first of
 * the order is always kept.  NaN logits count as -infinity, which is never drawn; where there is +infinity, only it is.  A row
 * without a logit above -infinity gets -1.  u outside [0, 1) is taken as the nearest in it, under 2^-40 as 0.  Weights are
 * summed as whole numbers of 2^-w of the largest, w = min(48, 63 - log2 of the row's length, rounded up), of which each above
 * 2^-1075 has one at least; rows of more than 8192 logits in stretches, each in units of its own largest weight, whose sums have one
 * of the row's units at least.  So results do not depend on any order.  min_p is compared with the weights themselves.
 */
typedef struct wc_sample_args {
  int32_t dtype;                  /* of the logits */
  int64_t n, m, v;                /* models, rows of each, logits of a row */
  const void* logits;             /* row r of model i at i * stride_n + (r / rows_inner) * stride_outer
                                     + (r % rows_inner) * stride_inner, unit stride over v */
  int64_t x_stride_n, x_stride_outer, x_stride_inner, x_rows_inner;
  const float* u;                 /* [n, m] */
  const float* temperature;       /* each of row r of model i at i * stride_n + r * stride_m */
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t temperature_stride_n, temperature_stride_m, top_k_stride_n, top_k_stride_m;
  int64_t top_p_stride_n, top_p_stride_m, min_p_stride_n, min_p_stride_m;
  int64_t* tokens;                /* [n, m] */
  void* workspace;                /* wc_sample_workspace_bytes(args), 16-byte aligned */
  int64_t workspace_bytes;
} wc_sample_args;

/* Bytes of workspace (0: none is needed), or -1 for sizes that wc_sample rejects. */
int64_t wc_sample_workspace_bytes(const wc_sample_args* args);

int32_t wc_sample(const wc_sample_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* WC_ANSWER_ABI_H */
