/*
 * What the requests of one batch bring of their own: low-rank adapters beside a projection that all of
 * them share, and the pick of each one's next token. C ABI, with the conventions of kernels.h: caller-owned
 * device memory, no allocation, shapes checked on the host, errors as llm_set_exit_on_error says. No
 * counterpart in the reference, which projects and samples one row (src/kernels.cuh:12-26).
 */
#ifndef LLM_AMD_BATCH_H
#define LLM_AMD_BATCH_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The adapters of a batch of sequences. A host struct; every pointer is device memory and is read when the
 * launched kernels run, so a captured graph follows the lengths and the choice of adapters.
 *
 * Sequence s has the rows q_start[s] .. q_start[s + 1] - 1 (from 0 to the call's n_tokens, not decreasing;
 * rows before q_start[0] and from q_start[n_seqs] on belong to no sequence and are left as they are), as
 * in PagedBatch, and the adapter adapter[s]; one outside [0, n_adapters) is none. Adapters of lower rank
 * than `rank` are filled up with zeros, in `a` or in `b` and finite in the other. */
typedef struct {
    const bf16 *a;          /* [n_adapters, rank, n_in], 16-byte aligned */
    const bf16 *b;          /* [n_adapters, n_out, rank], 16-byte aligned */
    const float *scale;     /* [n_adapters], or NULL: 1 */
    const int *q_start;     /* [n_seqs + 1] */
    const int *adapter;     /* [n_seqs] */
    int n_seqs;             /* at most 2^20, empty ones among them */
    int n_adapters;
    int rank;               /* a multiple of 8, at most 256 */
} LoraBatch;

/* out[t] = residual[t] + w x[t] + scale[a] b[a] (a[a] x[t]), a the adapter of row t's sequence; the last term
 * is not there for rows of sequences without one. w: [n_out, n_in], 16-byte aligned, or NULL: no product,
 * as beside a projection computed elsewhere. residual NULL: none; it may be out, row on row. lora NULL: no
 * adapters, and every row is computed. Otherwise nothing may overlap. x has rows x_stride elements apart (a multiple
 * of 8 up to 4194304, 16-byte aligned), out and residual rows out_stride and residual_stride apart, of any
 * alignment (multiples of 8 bytes are faster). n_in is a multiple of 8. Up to 2^20 rows, 2^20 of n_in and 2^22 of
 * n_out; a call that would take a launch of 2^31 threads or more is refused.
 * Products and sums are in 32 bits and rounded to bf16 once, at the end; scale a[a] x is kept to at least 16 bits
 * of its mantissa in front of b[a] (as a bf16 and the bf16 of what that leaves). The order of the sums depends on the
 * sizes and lengths alone. NaN and infinities of a row or an adapter reach no other row.
 * ws: lora_projection_workspace_floats() floats, 16-byte aligned, needing no preparation; calls that share it
 * must not overlap. */
void lora_projection_forward(bf16 *out, const bf16 *x, const bf16 *w, const bf16 *residual,
                             const LoraBatch *lora, float *ws, int n_tokens, int n_out, int n_in,
                             int64_t out_stride, int64_t x_stride, int64_t residual_stride,
                             hipStream_t stream);

/* Floats of ws that lora_projection_forward needs at most for these sizes and for any with fewer n_tokens or a
 * lower rank (0: no adapters): one workspace for the largest serves every call of the projection. */
size_t lora_projection_workspace_floats(int n_tokens, int n_out, int n_in, int rank);

/* Row r's next token into out[r]. The row's tokens stand in the order of their logits, largest first, equal ones
 * (0 and -0 among them) by lowest token; those of -inf or NaN are never taken. Their weights are
 * exp((x - max) / temperature), 1 for all of +inf where max is that, and of this order are left:
 *   the first top_k (all if that is not positive);
 *   of these the shortest part from the front whose weights add up to at least top_p of theirs, one token at
 *   least (all if top_p is 1 or more or NaN);
 *   of these the ones of weight min_p or more, one token at least (all if min_p is NaN).
 * out is the first of them whose running sum of weights passes u times their sum (the last of positive weight if
 * none does, the first if u is NaN), and logprob, if not NULL, ln of its weight over that sum. A temperature of 0
 * or less, or NaN: the first token, with logprob 0. A row of which nothing can be taken: -1, and -inf.
 * Weights and sums are in 64 bits, so that a pick does not depend on how they are added up (but for ties
 * within 2^-48 of the sum); logprob is rounded to 32.
 * temperature, top_p and min_p: [rows] floats, top_k: [rows] ints, each NULL where it is off (temperature: 1);
 * u: [rows], in [0, 1). Rows of logits are logits_stride elements apart, of any alignment. vocab: at most
 * 4194304. ws: sample_rows_workspace_floats() floats, 16-byte aligned, needing no preparation; calls that share it
 * must not overlap (NULL where the count is 0). */
void sample_rows_forward(int *out, float *logprob, const bf16 *logits, const float *temperature,
                         const int *top_k, const float *top_p, const float *min_p, const float *u,
                         float *ws, int rows, int vocab, int64_t logits_stride, hipStream_t stream);

/* Floats of ws that sample_rows_forward needs at most for these sizes and any smaller ones. */
size_t sample_rows_workspace_floats(int rows, int vocab);

#ifdef __cplusplus
}
#endif
#endif
