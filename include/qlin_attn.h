/*
 * qlin_attn.h -- C ABI of the attention operators in libqlin.so (MI355X, gfx950).
 *
 * What an attention layer of the engine does between its projections (proj3) and its
 * output projection (gate_mul_quant + gemm_i8): normalise and rotate queries and keys
 * and store keys and values in a paged cache, then attend -- over whole prompts, over
 * chunks of them, or for one new token of each sequence.  The rules of qlin.h hold: plain
 * device pointers, arguments checked before anything is launched, asynchronous launches on
 * `stream`, no allocation, status codes with the message in qlin_last_error(), and a
 * workspace of qlin_workspace_bytes() that calls overlapping in time must not share.
 *
 * Strides are in elements; the last axis (hd values) is contiguous.  Every 16-bit tensor
 * is 16-byte aligned with strides that are multiples of 8; int8 tensors have strides that
 * are multiples of 16.  Strides of tokens are at most 2^26, of heads and pages 2^31 - 16 (of an
 * int8 cache's scales 2^30 - 8); that of an axis of one is not looked at.  hd is 64, 128 or 256;
 * a key head has at most 64 query heads, a call at most 65536 query heads, 2^24 - 1 tokens and 65536
 * sequences, a sequence 2^30 keys.  scale is a positive number.  Lengths, page tables, slots and
 * positions are read on the device:
 *   - a slot below 0 or past the cache stores nothing (a padded row); the others of a call
 *     differ: what a slot given twice holds is of no one token;
 *   - kv_len below 0 counts as 0, above what the table's row holds as that;
 *   - a page outside 0 .. num_pages - 1 in front of a sequence's end makes NaN of every
 *     output that sees a key of it, and maybe of others of that sequence (no memory outside
 *     the cache is read);
 *   - a scale of an int8 cache that is not finite makes numbers of no output that sees its
 *     key; elsewhere infinities and NaN go through the formulas, but that an infinite fp16 value
 *     whose key weighs less than 2^-17 of its block's heaviest may make no number of its column
 *     (the weight is an fp16 number too, and may be zero);
 *   - row bounds (cu) are clamped to the rows there are, and query bounds that fall count as the
 *     highest before them.
 * Rows, heads and pages of what a call writes do not overlap, and it shares no byte with what the
 * call reads or else writes (q_out that is q and k_out that is k aside, with the same strides): such
 * calls are refused.  Tensors may lie between each other's rows, heads or pages; where they do so with
 * strides that are different but about the same length, over long axes, they are taken to overlap.
 */
#ifndef QLIN_ATTN_H
#define QLIN_ATTN_H

#include "qlin.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QLIN_I8 4

/* Keys and values of one layer in pages: element (page, token, head, i) of k lies at
 * k + page * k_page + token * k_token + head * k_head + i.  With int8 values, k_s / v_s
 * hold one fp32 scale of each (page, token, head): the value is code x scale. */
typedef struct qlin_paged_kv {
  void* k;
  int64_t k_page, k_token, k_head;
  void* v;
  int64_t v_page, v_token, v_head;
  float* k_s;
  int64_t ks_page, ks_token, ks_head;
  float* v_s;
  int64_t vs_page, vs_token, vs_head;
  int dtype;      /* QLIN_BF16, QLIN_F16 (the queries' type) or QLIN_I8 */
  int num_pages;
  int page;       /* tokens of a page: a power of two, 16 .. 1024 */
} qlin_paged_kv;

/* Arguments of qlin_qk_norm_rope. */
typedef struct qlin_rope {
  const void* q;               /* [T][q_heads][hd], `dtype` */
  int64_t q_token, q_head;
  const void* k;               /* [T][kv_heads][hd] */
  int64_t k_token, k_head;
  const void* v;               /* [T][kv_heads][hd], or NULL (no cache) */
  int64_t v_token, v_head;
  void* q_out;                 /* may be q itself, with its strides */
  int64_t qo_token, qo_head;
  void* k_out;                 /* rotated keys, may be k itself, with its strides; NULL: the cache only */
  int64_t ko_token, ko_head;
  const void* slots;           /* [T] places in the cache: page * page size + token; NULL: no cache */
  int slots_64;                /* 1: int64, 0: int32 */
  const void* pos;             /* [axes][T] positions */
  int64_t pos_axis, pos_token;
  int pos_64;
  const void* freqs;           /* [rot / 2] radians per position */
  int freqs_64;                /* 1: double, 0: float */
  const void* q_w;             /* RMSNorm weights [hd]; NULL: no norm */
  const void* k_w;
  int w_dtype;
  int one_plus;                /* scale by w + 1 */
  float eps;
  int T, q_heads, kv_heads, hd;
  int rot;                     /* leading values of a head that are turned: a multiple of 16 */
  int axes;                    /* 1 .. 3 */
  int sections[3];             /* frequencies of each axis; they add up to rot / 2 */
  int interleaved;             /* 0: runs of sections[a] frequencies; 1: axes take turns */
  int dtype;                   /* QLIN_BF16 or QLIN_F16 */
} qlin_rope;

/* Per head: y = x * rsqrt(mean(x^2) + eps) * (w + 1 or w) for queries and keys, then the
 * pairs (y[i], y[i + rot/2]) turned by pos[axis(i)][t] * freqs[i] (the angle in 64 bits),
 * rounded once to the output's type; keys and values to the cache's slots, as 16 bits or as
 * int8 codes round_half_away(y / s) with s = max(amax / 127, 1e-8) of the token's head.
 * cache NULL: keys go to k_out alone. */
int qlin_qk_norm_rope(const qlin_rope* args, const qlin_paged_kv* cache, void* stream);

/* Attention of packed prompts: sequence b's queries are rows cu_q[b] .. cu_q[b+1] - 1 of
 * q [T][q_heads][hd], its keys rows cu_k[b] .. of k, v [Tk][kv_heads][hd].
 * out = softmax(scale q k^T) v over all keys of the sequence, or where `causal` over the
 * keys j <= i + keys - queries for its query i.  Query head h uses key head
 * h / (q_heads / kv_heads).  A row that sees no key is zero; masked keys have no part in a
 * row whatever they hold.  Rows of no sequence are left as they were. */
int qlin_attn_prompt(const void* q, int64_t q_token, int64_t q_head,
                     const void* k, int64_t k_token, int64_t k_head,
                     const void* v, int64_t v_token, int64_t v_head,
                     const int* cu_q, const int* cu_k,
                     void* out, int64_t o_token, int64_t o_head,
                     int T, int Tk, int B, int q_heads, int kv_heads, int hd, int dtype,
                     float scale, int causal, void* workspace, size_t workspace_bytes, void* stream);

/* The same over the cache: sequence b's keys are the first kv_len[b] tokens of the pages
 * table[b][0 .. max_pages - 1] (its own queries' keys among them; of a table of no pages, which may be
 * NULL, no sequence has any). */
int qlin_attn_prompt_paged(const void* q, int64_t q_token, int64_t q_head, const qlin_paged_kv* cache,
                           const int* table, int64_t table_stride, int max_pages, const int* kv_len,
                           const int* cu_q, void* out, int64_t o_token, int64_t o_head,
                           int T, int B, int q_heads, int kv_heads, int hd, int dtype,
                           float scale, int causal, void* workspace, size_t workspace_bytes, void* stream);

/* One query per sequence, q and out [B][q_heads][hd]: attention over its kv_len[b] keys.
 * A sequence without keys gives zeros. */
int qlin_attn_decode(const void* q, int64_t q_seq, int64_t q_head, const qlin_paged_kv* cache,
                     const int* table, int64_t table_stride, int max_pages, const int* kv_len,
                     void* out, int64_t o_seq, int64_t o_head,
                     int B, int q_heads, int kv_heads, int hd, int dtype,
                     float scale, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QLIN_ATTN_H */
