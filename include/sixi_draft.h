/*
 * sixi_draft.h -- C ABI of the decision at the end of a speculative verify (gfx950): which drafted
 * tokens stay, and the token behind them, from the target's logits and given random numbers.
 *
 * Rows are the verify block's (sixi_attn.h): row 0 belongs to the anchor, row j to drafted token j-1,
 * and row j's logits are the target's for what follows it, i.e. for drafted token j.  With p_j the
 * softmax of row j's logits / temperature and q_j the distribution that token j was drawn from:
 *   token j stays if the ones before it do and u_j * q_j(d_j) < p_j(d_j)        (min(1, p / q));
 *   at the first that does not, the next token is drawn from max(p_j - q_j, 0), normalised;
 *   behind the last drafted token it is drawn from p.
 * A draw takes the smallest token i at which the running sum of the weights passes u_next * (their
 * sum).  So tokens are distributed as if drawn from p one by one, and the result is a function of
 * the inputs alone: sums run in 64 bits in a fixed order.
 *
 * Reference interfaces this replaces (file:line in the reference tree): the acceptance and
 * resampling of SpeculativeDecoder::step on the host (src/speculative/speculative.cpp:590-604), which
 * first reads the rows back.  `keep` is what sixi_gdn_params.snap takes, and kv_len[s] + keep[s] the
 * stream's cells afterwards.  Ownership and threading as in sixi_attn.h.
 */
#ifndef SIXI_DRAFT_H
#define SIXI_DRAFT_H

#include "sixi_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { SIXI_TYPE_BF16 = 30 }; /* ggml's id; logits and draft_probs only */

typedef struct sixi_draft_params {
    sixi_view logits;       /* [V, n_rows, S, 1] f32, f16 or bf16; elements contiguous          */
    sixi_view draft_probs;  /* [V, >= n_rows - 1, S, 1] f32, f16 or bf16: q; or data NULL: tokens
                               drafted without chance (q_j is 1 at d_j)                          */
    const int32_t* draft;   /* device: d_j of stream s at draft[s * draft_stride + j]; a token
                               outside [0, V) does not stay.  May be NULL if n_rows is 1         */
    int64_t draft_stride;
    const float* u;         /* device: u_j in [0, 1) at u[s * u_stride + j]; NULL as draft       */
    int64_t u_stride;
    const float* u_next;    /* device [S], in [0, 1)                                             */
    const float* temperature; /* device [S], or NULL (1).  0 or less: p is 1 at the largest logit,
                               the lowest such token                                             */
    const int32_t* q_len;   /* device [S]: rows of stream s, 1 + drafts (<= n_rows), or NULL      */
    int32_t* keep;          /* device [S]: rows that stay, 1 + tokens kept; 0 for q_len[s] <= 0   */
    int32_t* token;         /* device [S]: the next token; -1 for q_len[s] <= 0 or a row without
                               any weight                                                        */
    void* workspace;        /* device scratch of >= sixi_draft_workspace_bytes() bytes, 256-byte
                               aligned, no initialisation                                        */
    size_t workspace_bytes;
    int32_t flags;          /* reserved, must be 0                                               */
    int32_t reserved;
    void* stream;
} sixi_draft_params;

/* Decides every stream.  A logit of -inf or NaN has no weight (a sampler's filters strike tokens so);
 * +inf takes all.  A NaN temperature counts as 0.  If p - q leaves no weight, the draw is from p. */
int sixi_draft_verify(const sixi_draft_params* p);

int sixi_draft_workspace_bytes(const sixi_draft_params* p, size_t* bytes);

/* Host-side validation only: SIXI_OK or the error sixi_draft_verify returns, apart from the workspace's. */
int sixi_draft_validate(const sixi_draft_params* p);

#ifdef __cplusplus
}
#endif
#endif /* SIXI_DRAFT_H */
