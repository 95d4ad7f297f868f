/*
 * supra_kv.h - C ABI of attention over an 8-bit key/value cache on MI355X (gfx950): the norm and rotation
 * of new query and key rows, the cache written and read back, and attention over it.
 *
 * The reference keeps a context's projected K and V for a whole run in float32 (prepareContext,
 * app/models/dit.js:137-144) and attends to them at each of its steps (dit.js:180-185); it has no cache that
 * grows, no 8-bit values and no rotary positions. These calls hold such K and V in a quarter of the memory,
 * and let a sequence grow token by token.
 *
 * Same library and conventions as supra_attn.h (device pointers, offsets and strides in elements,
 * stream-ordered asynchronous calls on the current device, SA_OK or a negative SA_ERR_* status with
 * sa_last_error(), nothing allocated or synchronised inside a call, no memset recorded into a graph).
 * `dtype` names the type of the row tensors: SA_DT_F32, SA_DT_F16 or SA_DT_BF16 (supra_weights.h). Products,
 * sums and softmax statistics are float32 whatever it is, each output element rounded to it once.
 */
#ifndef SUPRA_KV_H
#define SUPRA_KV_H

#include "supra_attn.h"
#include "supra_weights.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms of queries and keys for each head, with the position rotation, in one pass ---- */
#define SA_NORM_NONE 0
#define SA_NORM_RMS 1  /* x / sqrt(mean(x^2) + eps) over the D elements of a head, times its weight */

#define SA_ROPE_HALF 0 /* pairs (i, i + rotary_dim/2) */
#define SA_ROPE_NEAR 1 /* pairs (2i, 2i + 1) */

/*
 * For each token t < T and head h, x = Q[t,h,:] (h < H) or K[t,h,:] (h < Hkv):
 *
 *   y = norm(x) * weight                             (float32 weight[D], NULL for ones)
 *   (y_a, y_b) <- rope_scale * (y_a cos f - y_b sin f, y_b cos f + y_a sin f),  f = positions[t] * inv_freq[i]
 *
 * for the i < rotary_dim/2 pairs (a, b) of the first rotary_dim elements; the others stay y. The angle f is
 * formed in float64, so far positions keep their precision; the rest is float32. Q[t,h,d] =
 * q[q_off + t*ldq + h*D + d], likewise k, q_out and k_out. Strides of 0 default to H*D (q) and Hkv*D (k).
 * rotary_dim 0 rotates nothing (positions and inv_freq may be NULL); Hkv 0 leaves k out, H 0 leaves q out. An
 * output may be its own input, rows and all (in place); otherwise outputs must not overlap what is read.
 * T = 0 is a call with nothing to do. D is even and at most 512.
 */
typedef struct sa_qk_rope_args {
  uint32_t struct_size;
  int32_t dtype; /* of q, k, q_out and k_out: SA_DT_F32, SA_DT_F16, SA_DT_BF16 */
  int32_t T;     /* tokens */
  int32_t H;     /* query heads */
  int32_t Hkv;   /* key heads */
  int32_t D;     /* head dim */
  int32_t rotary_dim; /* elements of a head that are rotated: even, 0..D */
  int32_t pairs;      /* SA_ROPE_HALF or SA_ROPE_NEAR */
  int32_t norm;       /* SA_NORM_* */
  float eps;          /* SA_NORM_RMS: >= 0 */
  float rope_scale;   /* factor of the rotated elements; 0 means 1 */
  const void* q;
  const void* k;
  int64_t q_off, k_off, ldq, ldk;
  void* q_out;
  void* k_out;
  int64_t qo_off, ko_off, ldqo, ldko;
  const float* q_weight;    /* [D] or NULL */
  const float* k_weight;    /* [D] or NULL */
  const double* inv_freq;   /* [rotary_dim / 2], radians per position */
  const int32_t* positions; /* [T] */
} sa_qk_rope_args;

int sa_qk_norm_rope(const sa_qk_rope_args* args, void* stream);

/* ---- the cache ---- */
#define SA_KV_BLOCK 32 /* tokens of a page: they share one scale for K and one for V in each head */

/*
 * `pages` pages of 32 tokens. The value of an element is its e4m3 code (OCP, largest value 448) times
 * 2^(e - 127), e the exponent byte of its page and head (E8M0). Powers of two scale without rounding, so a
 * page whose scale grows keeps every code that stays in e4m3's normal range bit for bit. Layout, that of the
 * matrix instructions' operands:
 *
 *   K: element (page, h, token t, d) at k[((page*Hkv + h)*(D/32) + d/32)*1024 + t*32 + d%32]
 *   V: element (page, h, token t, d) at v[((page*Hkv + h)*D + d)*32 + 16*((t/4)%2) + 4*(t/8) + t%4]
 *   exponents: k_scale[page*Hkv + h], v_scale[page*Hkv + h]
 *
 * k and v are 16-byte aligned and hold sa_kv_cache_bytes() bytes each, the exponents pages*Hkv bytes. They need no
 * initialisation: a page's bytes and exponents mean nothing until a write begins it.
 */
typedef struct sa_kv_cache {
  int32_t pages;
  int32_t Hkv;
  int32_t D; /* 64, 128 or 256 */
  int32_t reserved; /* 0 */
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
} sa_kv_cache;

/* Bytes of k, and of v: pages * Hkv * 32 * D, or a negative SA_ERR_* status. Host only. */
int64_t sa_kv_cache_bytes(int32_t pages, int32_t Hkv, int32_t D);

/*
 * The sequences of a call. Sequence b < B holds n = seq_len[b] tokens, token j in page
 * block_table[b*max_blocks + j/32] at place j%32. Its r = row_start[b+1] - row_start[b] rows in the call's row
 * tensors, from row row_start[b] on, are its last r tokens: positions n - r .. n - 1. row_start NULL stands for
 * max_rows rows of each sequence, b*max_rows on. All arrays are device memory, read by the kernels, so the host
 * needs only the bounds: T rows in the row tensors, at most max_rows of one sequence.
 *
 * What the arrays say is bounded by the kernels: lengths are taken within 0 .. 32*max_blocks, rows within
 * 0 .. max_rows and within the T rows, and a page id outside 0 .. pages-1 is a page that holds nothing (writes
 * to it are dropped, reads give zeros, attention passes its tokens over). Rows of the outputs that belong to no
 * sequence are left as they were. Pages may be shared by sequences that only read them; two sequences of one
 * write call, or two places of one sequence, must not write to the same page, and no two sequences of a call have a row in common (what such calls
 * leave is some mixture of both). A call's launch is shaped by the bounds: a batch of prompts and single tokens is
 * quicker as two calls, one with max_rows 1.
 */
typedef struct sa_kv_seqs {
  int32_t B;
  int32_t T;
  int32_t max_rows;
  int32_t max_blocks;
  const int32_t* row_start;   /* [B + 1] or NULL */
  const int32_t* seq_len;     /* [B] */
  const int32_t* block_table; /* [B, max_blocks] */
} sa_kv_seqs;

/* Rows of K and V: K[row,h,d] = k[k_off + row*ldk + h*D + d], likewise v; strides of 0 default to Hkv*D. */
typedef struct sa_kv_rows_args {
  uint32_t struct_size;
  int32_t dtype; /* of the rows: SA_DT_F32, SA_DT_F16, SA_DT_BF16 */
  sa_kv_cache cache;
  sa_kv_seqs seqs;
  void* k; /* read by sa_kv_write, written by sa_kv_read */
  void* v;
  int64_t k_off, v_off, ldk, ldv;
} sa_kv_rows_args;

/*
 * Quantises the rows into the cache (seq_len counts them already). A page's scale is the smallest power of two
 * that keeps its largest magnitude, new tokens and earlier ones of that sequence together, within 448 (2^-127
 * for zeros); values round to the nearest e4m3 value, ties to even. In a page that holds earlier tokens the
 * scale never shrinks, and where it grows their codes are brought to the new scale with the same rounding.
 * Infinities and NaN become NaN and do not count for the scale. Rows with no place (a negative position)
 * are dropped. Bytes of tokens behind the sequence's end are left as they were. The rows must not overlap the cache.
 */
int sa_kv_write(const sa_kv_rows_args* args, void* stream);

/* The rows' values from the cache, each rounded once to dtype (exact in float32, and in bfloat16 down to its
 * subnormals). Rows at negative positions and in pages that hold nothing are zeros. */
int sa_kv_read(const sa_kv_rows_args* args, void* stream);

/*
 * Attention over the cache: for each row i of sequence b and head h < H, with key head h / (H / Hkv),
 *
 *   o[i,h,:] = sum_j softmax_j(scale * q[i,h,:] . K[j,:]) V[j,:]
 *
 * over the sequence's tokens j < seq_len[b], or with `causal` those at or before the row's own position (the
 * rows are the sequence's last tokens, written before the call). Without `causal` the rows are queries of
 * their own, as of a cross-attention, and r may be more than n. A row that attends to nothing
 * is zeros. What lies behind a sequence's end, or behind a row's position, never enters its result, NaN codes
 * included. H is a multiple of Hkv.
 */
typedef struct sa_kv_attn_args {
  uint32_t struct_size;
  int32_t dtype; /* of q and o */
  sa_kv_cache cache;
  sa_kv_seqs seqs;
  int32_t H;
  int32_t causal;  /* 0 or 1 */
  float scale;     /* finite; magnitude below 2^127 */
  int32_t max_len; /* at least the longest seq_len, which shapes the launch (longer ones are still taken whole); 0: 32 * max_blocks */
  const void* q;
  void* o;
  int64_t q_off, o_off, ldq, ldo; /* Q[row,h,d] = q[q_off + row*ldq + h*D + d]; strides of 0: H*D */
  void* workspace;                /* device scratch, 16-byte aligned, when the call needs it */
  int64_t workspace_bytes;
} sa_kv_attn_args;

int sa_kv_attention(const sa_kv_attn_args* args, void* stream);

/* Scratch that sa_kv_attention needs for these arguments on the current device (0 where the keys of a row
 * are not split over workgroups), or a negative SA_ERR_* status. It holds no state between calls and needs no
 * initialisation; calls (and replays of graphs) that may run at the same time must not share one. Host only. */
int64_t sa_kv_attention_workspace_bytes(const sa_kv_attn_args* args);

/* How sa_kv_attention runs these arguments: query rows (tokens x heads of one key head) of a workgroup, and
 * workgroups that share the keys of those rows (their results are merged by a second launch where there is
 * more than one). SA_OK, or the status of a rejected call. Host only. */
int sa_kv_attention_shape(const sa_kv_attn_args* args, int32_t* rows, int32_t* splits);

#ifdef __cplusplus
}
#endif

#endif /* SUPRA_KV_H */
