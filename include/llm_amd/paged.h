/*
 * Serving operators over a paged KV cache, and the logits' penalties before a token is picked. C ABI,
 * with the conventions of kernels.h: caller-owned device memory, no allocation, shapes checked on the
 * host, errors as llm_set_exit_on_error says. No counterpart in the reference, whose cache is one
 * contiguous row of positions for one sequence (src/forward.cuh:6-25): these take many sequences, each
 * with any number of new tokens, over a pool of pages. They compute in 32 bits (angles in 64) and round
 * to bf16 once, at the end; the attention's weights are its one other rounding (see there).
 */
#ifndef LLM_AMD_PAGED_H
#define LLM_AMD_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A batch of sequences over a pool of pages. A host struct; every pointer is device memory and is read
 * when the launched kernels run, so a captured graph follows the lengths and the table as they change.
 *
 * Sequence s has the new tokens of rows q_start[s] .. q_start[s + 1] - 1 (from 0 to the call's n_tokens, not
 * decreasing; rows before q_start[0] and from q_start[n_seqs] on belong to no sequence and are left as they
 * are), and kv_len[s] tokens in the cache once the new ones are in (more than 2^30 count as 2^30): its i-th
 * new row has the position kv_len[s] - (q_start[s + 1] - q_start[s]) + i. Position p lies in page page_table[s, p / page_size] of the
 * pool, at slot p % page_size; element d of its kv head h is at
 * page * page_stride + slot * slot_stride + h * head_stride + d of the key and of the value cache.
 * Positions past the table's row, and those whose page is outside [0, n_pages), are not there: they are
 * neither written nor seen. */
typedef struct {
    bf16 *key_cache;        /* 16-byte aligned */
    bf16 *value_cache;
    int64_t page_stride;    /* elements, multiples of 8, not negative; to be written into: at least head_dim */
    int64_t slot_stride;    /* at least head_dim, at most 2^26 */
    int64_t head_stride;    /* like page_stride */
    const int *page_table;  /* [n_seqs, table_pages] */
    const int *q_start;     /* [n_seqs + 1] */
    const int *kv_len;      /* [n_seqs] */
    int n_seqs;
    int n_pages;
    int page_size;
    int table_pages;
    int n_kv_heads;
    int head_dim;           /* 64, 128 or 256 */
} PagedBatch;

/* How rope_frequencies stretches the rotation past the trained length. */
enum { ROPE_PLAIN = 0, ROPE_LINEAR = 1, ROPE_YARN = 2 };

/* Radians per position of the rotary_dim / 2 rotated pairs, theta^(-2j / rotary_dim), into inv_freq (host
 * memory), and the factor of cos and sin as the result (0 after an error). ROPE_LINEAR: all of them
 * divided by `factor`. ROPE_YARN: pairs that turn less than once over `trained` positions are divided by
 * factor, those that turn more than 32 times are left, with a ramp over the pairs between; the result is
 * 0.1 ln(factor) + 1 instead of 1. `trained` is read by ROPE_YARN alone. */
float rope_frequencies(double *inv_freq, int rotary_dim, double theta, int kind, double factor,
                       int trained);

/* qk_norm_rope_rows for a paged cache. Of every row of a sequence: each head of q and k is divided by its
 * RMS and multiplied by q_norm_w / k_norm_w (NULL: left as it is), its first rotary_dim elements are
 * rotated by position * inv_freq[j], cos and sin times rope_scale, q goes to q_out and k and v to the
 * row's place in the caches (q_out alone where the position is not there, negative ones included).
 * Pair j is the elements j and j + rotary_dim / 2 (interleaved 0) or 2j and 2j + 1 (1). inv_freq: device,
 * [rotary_dim / 2] doubles. q, k and v have rows of heads * head_dim elements q_stride, k_stride and
 * v_stride apart (multiples of 8), as slices of one q/k/v projection have; q_out likewise. q_out may be q,
 * row on row; nothing else may overlap. rotary_dim is a multiple of 16, at most head_dim. Two rows with one place in
 * the cache leave either's k and v there, head by head. */
void qk_norm_rope_paged(bf16 *q_out, const bf16 *q, const bf16 *k, const bf16 *v,
                        const bf16 *q_norm_w, const bf16 *k_norm_w, const double *inv_freq,
                        const PagedBatch *batch, int n_tokens, int n_heads, int rotary_dim,
                        int interleaved, float eps, float rope_scale, int64_t q_out_stride,
                        int64_t q_stride, int64_t k_stride, int64_t v_stride, hipStream_t stream);

/* Attention of every new row over its sequence's cache: the row at position p sees the positions
 * max(0, p - window + 1) .. p that are there (window 0: from 0 on), softmax(q . k * scale) over them, and
 * out is the weighted sum of their values. A row that sees nothing, or only scores of -inf, gives
 * zeros. What lies in the caches at positions that a row does not see, NaN and infinities included, does
 * not reach it. A value that it sees and that is infinite makes its element infinite, or no number where its weight
 * falls below the range of 32 bits; finite values overflow where their size times 2^8 times the number of
 * positions passes that range. Query head h reads kv head h / (n_heads / n_kv_heads). Rows of q and out are
 * q_stride and out_stride elements apart; out must not overlap anything. scale > 0.
 * Scores, weights and sums are in 32 bits; in front of the values the weights are rounded to bf16. What that leaves
 * is added back where rows are few, since there the bytes of the cache take longer than both products: in sequences
 * of at most 32 rows x heads per kv head, and in all of them where max_q_len expects no more. It is not where n_tokens,
 * n_seqs and max_q_len leave room for no such sequence (one sequence of which more is expected, for instance), nor in
 * what a workgroup computes (few rows, some keys) if a part of it is infinite or no number.
 * max_q_len and max_kv_len say how many new rows and how many cached tokens a sequence is expected to have at
 * most: the split of the work goes by them. Longer sequences are computed all the
 * same, more slowly. How the work is split changes the order of the sums and with it the last bits.
 * ws: attention_paged_workspace_floats() floats, 16-byte aligned, needing no preparation; calls that share
 * it must not overlap (NULL where the count is 0). */
void attention_paged_forward(bf16 *out, const bf16 *q, const PagedBatch *batch, float *ws,
                             int n_tokens, int n_heads, int max_q_len, int max_kv_len, int window,
                             float scale, int64_t out_stride, int64_t q_stride, hipStream_t stream);

/* Floats of ws that attention_paged_forward needs at most for these sizes and for any with fewer n_tokens, n_seqs,
 * max_q_len or max_kv_len (the heads being the same): one workspace for the largest serves every call. */
size_t attention_paged_workspace_floats(int n_tokens, int n_seqs, int n_heads, int n_kv_heads,
                                        int head_dim, int max_q_len, int max_kv_len);

/* Logits as a sampler wants them, one row per sequence; in this order, in 32 bits, rounded once:
 *   a token among the row's token_len tokens: x = x > 0 ? x / repetition : x * repetition;
 *   a token n > 0 times among those from prompt_len on: x -= frequency * n + presence;
 *   a token among the row's bias_len bias_tokens: x += its bias (of several entries the last counts);
 *   a token whose bit is 0 in `allowed` (bit t % 32 of word t / 32): x = -inf, whatever it was.
 * tokens: [rows, token_stride]; bias_tokens and bias: [rows, bias_stride]; allowed: [rows, allowed_stride]
 * words. prompt_len and token_len are counts within the row's token_stride entries, and bias_len within
 * bias_stride (at most 2^22): what is outside is cut off. Tokens outside [0, vocab) are passed over. repetition, frequency and
 * presence: [rows], each NULL where it is off; tokens NULL: no history; bias_tokens NULL: no biases;
 * allowed NULL: no mask; prompt_len NULL: no prompt; bias_len NULL: all bias_stride entries. Rows of
 * logits and out are logits_stride and out_stride elements apart; out may be logits. */
void logits_penalty_forward(bf16 *out, const bf16 *logits, const int *tokens, const int *prompt_len,
                            const int *token_len, const float *repetition, const float *frequency,
                            const float *presence, const int *bias_tokens, const float *bias,
                            const int *bias_len, const uint32_t *allowed, int rows, int vocab,
                            int token_stride, int bias_stride, int allowed_stride,
                            int64_t out_stride, int64_t logits_stride, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
