/*
 * qlin_candidates.h -- C ABI of a decode step of several candidates of one prompt in
 * libqlin.so (MI355X, gfx950).
 *
 * The engine answers a prompt with several candidates at once: one prefill, then steps of
 * one token of each (generate_batch, sample_batch).  Beside the linears and the attention
 * operators such a step takes attention that reads a shared prompt once for all of its
 * candidates, and what lies between the vocabulary head and the next token: penalties,
 * biases and masks on the logits, and the draw.  The rules of qlin.h hold: plain device
 * pointers, arguments checked before anything is launched, asynchronous launches on
 * `stream`, no allocation, status codes with the message in qlin_last_error(), and a
 * workspace of qlin_workspace_bytes() that calls overlapping in time must not share.
 */
#ifndef QLIN_CANDIDATES_H
#define QLIN_CANDIDATES_H

#include "qlin_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One query per sequence, q and out [B][q_heads][hd].  Sequences come in G groups: group g's are
 * cu_seq[g] .. cu_seq[g+1] - 1, and all of them see the first prefix_len[g] tokens of pages
 * prefix_table[g][0 .. max_prefix_pages - 1], which are read from memory once for the group (by tiles of 16 to
 * 128 query rows, chosen by the average group, that meet in the L2 caches), and then their own first
 * kv_len[b] tokens of pages table[b][0 .. max_pages - 1] (the new one among them; a table of no pages may
 * be NULL):
 * out = softmax(scale q k^T) v over both.  Prefix and own keys lie in one cache.  A sequence without keys
 * gives zeros; sequences of no group (behind cu_seq[G]) are left as they were.  What qlin_attn.h
 * states of strides, limits, lengths, pages and scales holds here too; cu_seq is clamped to the sequences
 * there are, and bounds that fall count as the highest before them.  Whatever sizes a query's values have and
 * however many sequences see a key: over int8 keys a weight of the softmax may be off by 2^-16 of itself more
 * than over 16-bit ones; with fp16 values one as far as 18 octaves below the heaviest of its 32 keys is rounded
 * to fp16's 11 bits, a lighter one is off by at most 2^-29 of that heaviest.
 * A call's query values (B x q_heads x hd) are at most about 2^24, whatever groups the sequences are in, as the
 * workspace holds 32-bit sums of each twice, and those of a cut (a tile of up to 128 rows of each key head). */
int qlin_attn_decode_shared(const void* q, int64_t q_seq, int64_t q_head, const qlin_paged_kv* cache,
                            const int* prefix_table, int64_t prefix_table_stride, int max_prefix_pages,
                            const int* prefix_len, const int* cu_seq, int G,
                            const int* table, int64_t table_stride, int max_pages, const int* kv_len,
                            void* out, int64_t o_seq, int64_t o_head,
                            int B, int q_heads, int kv_heads, int hd, int dtype,
                            float scale, void* workspace, size_t workspace_bytes, void* stream);

/* Arguments of qlin_logits_process.  A number of each row is a vector [B], or NULL and one number for all. */
typedef struct qlin_logits {
  const void* logits;          /* [B][V], `dtype`, rows at any element's address */
  int64_t logits_row;          /* row strides are in elements */
  void* out;                   /* [B][V], `out_dtype`; may be logits itself, with its dtype and stride */
  int64_t out_row;
  const void* tokens;          /* [B][history] tokens of each row so far, the prompt's first; NULL: none */
  int64_t tokens_row;
  const int* lens;             /* [B] how many of them there are; NULL: history of each */
  const int* prompt_lens;      /* [B] how many of those are the prompt's; NULL: none */
  const float* repetition;     /* [B] */
  const float* presence;
  const float* frequency;
  const int* bias_ids;         /* [B][biases] tokens */
  int64_t bias_ids_row;
  const float* bias;           /* [B][biases] what is added to theirs */
  int64_t bias_row;
  const void* mask;            /* allowed tokens: bits [B][(V + 31) / 32] of int32 words, the lowest first, or
                                  bytes [B][V]; a row stride of 0 is one mask for all rows; NULL: all */
  int64_t mask_row;
  int tokens_64;               /* 1: int64, 0: int32 */
  int mask_bytes;
  int B, V, history, biases;
  int dtype, out_dtype;        /* QLIN_BF16, QLIN_F16 or QLIN_F32 */
  float repetition_all, presence_all, frequency_all;
} qlin_logits;

/* What a token's logit x becomes, in 32 bits, each step rounded once, in this order:
 *   x > 0 ? x / repetition : x * repetition    where the row's history holds the token;
 *   x - frequency * c - presence               where it comes c > 0 times behind the prompt;
 *   x + bias                                   where the row's bias_ids hold it (of an id that is given more
 *                                              than once the last counts);
 *   -inf                                       where the mask does not allow it;
 * and then the output's type.  Ids outside 0 .. V - 1 (padding) count for nothing; lens is clamped to 0 ..
 * history.  A repetition that is one number for all is a positive one.  Infinities and NaN go through the
 * formulas.  out shares no byte with what the call reads (the logits themselves aside). */
int qlin_logits_process(const qlin_logits* args, void* stream);

/* One token of each row of logits [B][V], into tokens [B] (int64 or int32), with a uniform number u[b] of
 * 0 <= u < 1.  Of the row's top_k (1 .. 128) largest logits x_0 >= x_1 >= ..., equal ones by their index, with
 * weights w_i = exp((x_i - x_0) / temperature), those are kept that have less than top_p of the weights' sum
 * in front of them and weigh at least min_p (x_0 always), and the first is drawn with which the sum of the
 * kept exceeds u times theirs.  Temperature 0: the largest, of equal ones the lowest index, whatever u is (a
 * vector's negative numbers and NaN count as 0).  Sums and weights are of 64 bits.  logprobs [B] (or NULL):
 * x - log sum exp of the row's logits, at the token.
 * A logit of -inf or NaN is never drawn and has no part in a sum; a row of nothing else gives token -1 and -inf.
 * Infinite logits share the row among themselves, at temperature 0 too.  A number of each row is a vector [B],
 * or NULL and one number for all.  What the call writes shares no byte with what it reads. */
int qlin_sample(const void* logits, int dtype, int64_t logits_row, int B, int V, int top_k, const float* u,
                const float* temperature, float temperature_all, const float* top_p, float top_p_all,
                const float* min_p, float min_p_all, void* tokens, int tokens_64, float* logprobs,
                void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QLIN_CANDIDATES_H */
