/*
 * pkda_serve_gfx950.h -- C ABI of the serving operators beside the PKDA layers
 * (gfx950): a paged key/value cache, the attention that reads it, the sampling
 * of the next token and the verification of drafted ones.  They are in libpkda_gfx950.so; conventions,
 * status codes, dtypes and pkda_last_error() are those of pkda_gfx950.h.
 *
 * The paged cache.  Keys and values live in two pools of pages,
 * [num_pages, page_size, kv_heads, head_dim] each, every page dense, pages
 * k_page_stride / v_page_stride elements apart.  Position p of sequence n is
 * row p % page_size of page page_table[n][p / page_size].  A sequence holds
 * seq_lens[n] positions, its new tokens among them: with cu_seqlens
 * (int32 [num_seqs + 1], device) tokens cu[n] .. cu[n+1] - 1 are its last
 * cu[n+1] - cu[n] positions; without, every sequence has one new token.
 *
 * What a caller's device data can say wrong stays inside the buffers: a length
 * past the table's row is cut to it, document bounds are clamped to the packed
 * length and cu[0] counts as 0, a page number outside the pool holds nothing
 * (nothing is stored there, its positions are masked), a token of no sequence
 * (past cu[num_seqs], or before its sequence's position 0) has no key.  Bounds
 * that fall name no sequences: which of the sequences' rows are written, and
 * what the tokens' outputs hold, is undefined then.
 */
#ifndef PKDA_SERVE_GFX950_H
#define PKDA_SERVE_GFX950_H

#include "pkda_gfx950.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PKDA_SERVE_ABI_VERSION 2

int pkda_serve_abi_version(void);
/* sizeof() of each argument struct below. */
int64_t pkda_serve_args_size(int which);
enum pkda_serve_args_kind {
  PKDA_SERVE_ARGS_APPEND = 0,
  PKDA_SERVE_ARGS_ATTENTION = 1,
  PKDA_SERVE_ARGS_SAMPLE = 2,
  PKDA_SERVE_ARGS_STORE = 3,
  PKDA_SERVE_ARGS_ATTENTION_FP8 = 4,
  PKDA_SERVE_ARGS_PREFIX = 5,
  PKDA_SERVE_ARGS_VERIFY = 6
};

/* ---------------------------------------------------------------------------
 * Append: the new tokens' keys and values into the cache, with the rotary
 * position embedding of keys (and queries) on the way.
 *
 * The first rotary_dim channels of a head at position p turn by the angles of
 * row p of cos / sin ([rope_rows, rotary_dim / 2] FP32):
 *   (a, b) -> (a cos - b sin, b cos + a sin)
 * with (a, b) = channels (c, c + rotary_dim / 2), or (2c, 2c + 1) when
 * interleaved; FP32, rounded once.  Channels past rotary_dim, values, and with
 * cos == NULL everything, are copied as they are.  q_out [num_tokens, q_heads,
 * head_dim] is dense; rows of tokens without a position are zeros.
 * Concurrent writers of one row (sequences that share a page being written)
 * are the caller's error.
 * ------------------------------------------------------------------------- */
typedef struct pkda_paged_append_args {
  int32_t struct_size;  /* sizeof(pkda_paged_append_args) */
  int32_t dtype;        /* pkda_dtype of q, k, v, the pools */
  int32_t num_seqs, num_tokens, q_heads, kv_heads, head_dim; /* q_heads 0: no q */
  int32_t page_size, max_pages; /* max_pages: pages of a table row; page_size * max_pages <= 2^30 */
  int64_t num_pages;
  int64_t table_stride;         /* elements between table rows */
  const int32_t* cu_seqlens;    /* [num_seqs + 1] or NULL (num_tokens == num_seqs) */
  const int32_t* seq_lens;      /* [num_seqs], the new tokens included */
  const int32_t* page_table;    /* [num_seqs, max_pages] */
  const void* q;                /* [num_tokens, q_heads, head_dim], tokens q_stride elements apart */
  const void* k;                /* [num_tokens, kv_heads, head_dim] */
  const void* v;
  int64_t q_stride, k_stride, v_stride; /* multiples of 16 bytes */
  void* q_out;
  void* k_pages;
  void* v_pages;
  int64_t k_page_stride, v_page_stride; /* elements; multiples of 16 bytes */
  const float* cos;             /* or NULL: no rotation */
  const float* sin;
  int32_t rotary_dim;           /* a multiple of 16, <= head_dim */
  int32_t interleaved;
  int64_t rope_rows;            /* >= max_pages * page_size */
} pkda_paged_append_args;

int pkda_paged_append(const pkda_paged_append_args* args, void* stream);

/* ---------------------------------------------------------------------------
 * Attention of the new tokens over the cache, which holds their own keys and
 * values already.  Query head h reads key/value head h / (q_heads / kv_heads).
 * Token t at position p(t) sees positions 0 .. p(t):
 *   s = scale q . K[pos];  o = sum softmax(s) V;  lse = log sum exp(s)
 * Scores, softmax statistics and sums are FP32 (BF16: the probabilities are
 * rounded to BF16 as operands of the product with V, each output rounded
 * once).  A token without keys has o = 0 and lse = -inf.
 * ------------------------------------------------------------------------- */
typedef struct pkda_paged_attention_args {
  int32_t struct_size;
  int32_t dtype;
  int32_t num_seqs, num_tokens, q_heads, kv_heads, head_dim;
  int32_t page_size, max_pages;
  int64_t num_pages;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* seq_lens;
  const int32_t* page_table;
  const void* q;                /* tokens q_stride elements apart */
  int64_t q_stride;
  const void* k_pages;
  const void* v_pages;
  int64_t k_page_stride, v_page_stride;
  float scale;
  void* o;                      /* [num_tokens, q_heads, head_dim] dense */
  float* lse;                   /* [num_tokens, q_heads] */
  float* workspace;             /* pkda_paged_attention_workspace() floats */
} pkda_paged_attention_args;

/* Floats of workspace the call needs at most, from its sizes alone (no pointer
 * is looked at, cu_seqlens neither: where num_tokens == num_seqs it is enough
 * with cu_seqlens and without); < 0 for sizes the call refuses. */
int64_t pkda_paged_attention_workspace(const pkda_paged_attention_args* args);
int pkda_paged_attention(const pkda_paged_attention_args* args, void* stream);

/* ---------------------------------------------------------------------------
 * The next token of each row of logits, with temperature, top-k, top-p and
 * min-p, from given Gumbel numbers.
 *
 * Per row, with l in FP32, m = max l, z_i = (l_i - m) / temperature,
 * w_i = e^{z_i}, tokens in order of l descending, index ascending:
 *   K = the first top_k tokens (all of them when top_k <= 0)
 *   P = those tokens of K before which K holds less than top_p sum_K w
 *       (all of them when top_p >= 1; the first token is always in)
 *   M = those with w_i >= min_p
 *   token = the lowest index that maximises z_i + noise_i over K, P and M
 * temperature <= 0 takes the first token of the order.  logprob is the token's
 * log softmax(l): unfiltered, at temperature 1.  NaN and -inf logits are never
 * taken; +inf counts as the largest finite number.  A row without any other
 * logit has token -1 and logprob -inf.  Sums are FP32 or wider in a fixed
 * order.
 * ------------------------------------------------------------------------- */
typedef struct pkda_sample_args {
  int32_t struct_size;
  int32_t dtype;                /* of logits */
  int32_t rows, vocab;
  const void* logits;           /* [rows, vocab], rows logits_stride elements apart */
  int64_t logits_stride;
  const float* noise;           /* [rows, vocab], rows noise_stride elements apart */
  int64_t noise_stride;
  const float* temperature;     /* [rows], or NULL: temperature_all for every row */
  const int32_t* top_k;         /* likewise */
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int32_t top_k_all;            /* 0: off */
  float top_p_all;              /* 1: off */
  float min_p_all;              /* 0: off */
  int32_t* token;               /* [rows] */
  float* logprob;               /* [rows] */
} pkda_sample_args;

int pkda_sample(const pkda_sample_args* args, void* stream);

/* ---------------------------------------------------------------------------
 * A cache of 8-bit floats: pools [num_pages, page_size, kv_heads, head_dim] of
 * E4M3 codes (4 exponent bits, 3 mantissa bits, no infinity), and for each 32
 * channels of a row a scale 2^(e - 127) held as the byte e,
 * [num_pages, page_size, kv_heads, head_dim / 32], pages k_scale_stride /
 * v_scale_stride bytes apart.  A number is code * scale, exact in BF16 and FP32 for
 * the scales that the store writes, bytes 10 .. 246; what others stand for where a
 * sequence has a position is undefined.  head_dim 64 or 128.
 *
 * Store: pkda_paged_append with, on the way, the norms of query and key heads,
 * before the rotation (NULL: none):
 *   x <- x (mean x^2 + eps)^(-1/2) w      over the head's channels, in FP32
 * into a cache of the activations' type (cache_dtype == dtype) or of 8-bit
 * floats (PKDA_CACHE_FP8).  There a block's scale is the smallest of 2^-117 ..
 * 2^119 by which its largest finite magnitude is at most 448, and a code the
 * nearest (ties to even) of the FP32 number over the scale, held to +-448; NaN
 * and infinities are stored as NaN.
 * ------------------------------------------------------------------------- */
#define PKDA_CACHE_FP8 2

typedef struct pkda_paged_store_args {
  int32_t struct_size;  /* sizeof(pkda_paged_store_args) */
  int32_t dtype;        /* pkda_dtype of q, k, v */
  int32_t num_seqs, num_tokens, q_heads, kv_heads, head_dim; /* as pkda_paged_append_args */
  int32_t page_size, max_pages;
  int64_t num_pages;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* seq_lens;
  const int32_t* page_table;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_stride, k_stride, v_stride;
  void* q_out;
  void* k_pages;
  void* v_pages;
  int64_t k_page_stride, v_page_stride; /* elements of the cache */
  const float* cos;
  const float* sin;
  int32_t rotary_dim;
  int32_t interleaved;
  int64_t rope_rows;
  int32_t cache_dtype;  /* dtype, or PKDA_CACHE_FP8 */
  int32_t norm_dtype;   /* pkda_dtype of q_norm, k_norm */
  const void* q_norm;   /* [head_dim] or NULL */
  const void* k_norm;
  float eps;
  uint8_t* k_scales;    /* PKDA_CACHE_FP8: aligned to head_dim / 32 bytes, strides too */
  uint8_t* v_scales;
  int64_t k_scale_stride, v_scale_stride;
} pkda_paged_store_args;

int pkda_paged_store(const pkda_paged_store_args* args, void* stream);

/* pkda_paged_attention over a cache of 8-bit floats; q and o are of dtype. */
typedef struct pkda_paged_attention_fp8_args {
  int32_t struct_size;
  int32_t dtype;
  int32_t num_seqs, num_tokens, q_heads, kv_heads, head_dim;
  int32_t page_size, max_pages;
  int64_t num_pages;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* seq_lens;
  const int32_t* page_table;
  const void* q;
  int64_t q_stride;
  const void* k_pages;
  const void* v_pages;
  int64_t k_page_stride, v_page_stride; /* bytes; multiples of 16 */
  float scale;
  void* o;
  float* lse;
  float* workspace;             /* pkda_paged_attention_fp8_workspace() floats */
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  int64_t k_scale_stride, v_scale_stride;
} pkda_paged_attention_fp8_args;

int64_t pkda_paged_attention_fp8_workspace(const pkda_paged_attention_fp8_args* args);
int pkda_paged_attention_fp8(const pkda_paged_attention_fp8_args* args, void* stream);

/* ---------------------------------------------------------------------------
 * Attention of a batch in groups of sequences that share their first positions,
 * over a cache of the activations' type or of 8-bit floats.  Sequences
 * cu_groups[g] .. cu_groups[g+1] - 1 (int32 [num_groups + 1], device; cu_groups[0]
 * counts as 0, bounds are clamped to num_seqs, sequences past the last share
 * nothing) hold the same keys and values at positions 0 .. prefix_lens[g] - 1,
 * in the same pages or in copies: from the pages of which of the sequences that
 * hold a position it is read is not said.  A sequence of fewer positions than the
 * prefix (a slot that is finished, of none) sees what it holds of it; the others see
 * all of it, wherever that one stands in the group and whatever its row of the table
 * says past its length.  The result is that of pkda_paged_attention.
 * ------------------------------------------------------------------------- */
typedef struct pkda_paged_prefix_args {
  int32_t struct_size;
  int32_t dtype;
  int32_t num_seqs, num_tokens, q_heads, kv_heads, head_dim;
  int32_t page_size, max_pages;
  int64_t num_pages;
  int64_t table_stride;
  const int32_t* cu_seqlens;
  const int32_t* seq_lens;
  const int32_t* page_table;
  const void* q;
  int64_t q_stride;
  const void* k_pages;
  const void* v_pages;
  int64_t k_page_stride, v_page_stride;
  float scale;
  void* o;
  float* lse;
  float* workspace;             /* pkda_paged_prefix_workspace() floats */
  const uint8_t* k_scales;      /* or NULL: a cache of dtype */
  const uint8_t* v_scales;
  int64_t k_scale_stride, v_scale_stride;
  const int32_t* cu_groups;     /* [num_groups + 1] */
  const int32_t* prefix_lens;   /* [num_groups] */
  int32_t num_groups;
} pkda_paged_prefix_args;

int64_t pkda_paged_prefix_workspace(const pkda_paged_prefix_args* args);
int pkda_paged_prefix_attention(const pkda_paged_prefix_args* args, void* stream);

/* ---------------------------------------------------------------------------
 * Verification of drafted tokens, from given random numbers.
 *
 * Rows cu_seqlens[n] .. cu_seqlens[n+1] - 1 are those of sequence n (bounds
 * clamped and cu_seqlens[0] 0 as above): row j of them holds the target's logits
 * after the sequence's first j drafts, and drafts[row], its uniform number and
 * its draft_logits (those the draft was drawn from) are of the draft after that
 * place; the last row has none, whatever its entries hold.  With
 *   p = softmax(l / temperature),  q = softmax(draft l / temperature), or 1 at the
 *   draft and 0 elsewhere where draft_logits is NULL,
 * drafts are accepted in turn while  uniform q(d) < p(d).  The token after the
 * accepted ones is the lowest index that maximises log r + noise over r > 0, r =
 * max(p - q, 0) in the row of the first draft that is not accepted (p where that
 * is nowhere positive), p in the last row and in one whose draft is outside the
 * vocabulary, where nothing was drawn from q.  temperature <= 0 accepts a draft
 * that is the lowest index of the largest logit, and takes that as the next token.
 * An infinite temperature makes p and q even over what has a logit.
 *
 * NaN and -inf logits have p = 0 (q = 0); +inf counts as the largest finite
 * number.  A draft outside the vocabulary (none) is not accepted.  A row without
 * any other logit accepts nothing and its token is -1.
 * tokens[row] is the row's draft where that was accepted, the next token in the
 * row after those, and -1 in the others (and in rows of no sequence).
 * ------------------------------------------------------------------------- */
typedef struct pkda_verify_args {
  int32_t struct_size;
  int32_t dtype;                /* of logits and draft_logits */
  int32_t rows, vocab, num_seqs;
  const void* logits;           /* [rows, vocab], rows logits_stride elements apart */
  int64_t logits_stride;
  const void* draft_logits;     /* likewise, or NULL */
  int64_t draft_stride;
  const int32_t* drafts;        /* [rows] */
  const float* uniform;         /* [rows], in [0, 1) */
  const float* noise;           /* [num_seqs, vocab] Gumbel numbers */
  int64_t noise_stride;
  const int32_t* cu_seqlens;    /* [num_seqs + 1] */
  const float* temperature;     /* [num_seqs], or NULL: temperature_all */
  float temperature_all;
  int32_t* tokens;              /* [rows] */
  int32_t* accepted;            /* [num_seqs] */
  float* workspace;             /* pkda_verify_workspace() floats */
} pkda_verify_args;

int64_t pkda_verify_workspace(const pkda_verify_args* args); /* from the sizes alone; < 0: refused */
int pkda_verify(const pkda_verify_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PKDA_SERVE_GFX950_H */
