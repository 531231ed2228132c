/*
 * bigsmall_draft.h — C ABI of the verification of drafted tokens
 * (libbigsmall_hip.so). No reference counterpart.
 *
 * As in bigsmall_hip.h: plain pointers and sizes, `stream` a hipStream_t as
 * void*, the call asynchronous on it, BS_DEV_* bits OR-ed into *d_status (may be
 * NULL). It allocates nothing, does not synchronise, keeps no state and may be
 * captured into a graph.
 */
#ifndef BIGSMALL_DRAFT_H
#define BIGSMALL_DRAFT_H

#include <stdint.h>

#include "bigsmall_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define BS_DRAFT_F32 0
#define BS_DRAFT_BF16 1
#define BS_DRAFT_F16 2
#define BS_DRAFT_MOST 1024 /* drafts of a sequence */

/* Row r of p is the target's distribution after row r's token, row r of q the
 * draft model's, draft[r] the token proposed to follow it. Drafts are taken by p
 * and q as they are: tokens follow p only if their rows add up to 1. Sequence b has
 * rows cu[b] .. cu[b + 1] - 1, one more than drafts (its last row of q, draft and
 * accept is not read); one without rows takes no part. */
typedef struct {
    const void *p, *q;     /* [n_rows][vocab], rows p_stride and q_stride elements apart; q may be NULL */
    const int64_t *draft;  /* [n_rows] */
    const float *accept;   /* [n_rows] random numbers in [0, 1) */
    const int32_t *cu;     /* [n_seqs + 1] */
    const float *pick;     /* [n_seqs] random numbers in [0, 1) */
    int64_t *tokens;       /* [n_seqs][max_drafts + 1]: drafts taken, the token drawn, then -1 */
    int32_t *counts;       /* [n_seqs] tokens of a sequence */
    int64_t p_stride, q_stride;
    uint32_t type, n_rows, vocab, n_seqs, max_drafts;
} bs_draft_batch;

/* Draft x is taken while accept * q[x] < p[x] (accept < p[x] without q); then one token is drawn: where a draft was
 * refused from w = max(p - q, 0) of its row (without q: p, the draft's own weight 0), after the last one from w = p. It is
 * the first at which the sum of w up to it exceeds pick times the sum of all, in 64 bits. Weights that are no numbers or
 * negative are 0, infinite ones the largest f32. If no weight is above 0, w is p; if none is then, the token is 0 and
 * BS_DEV_ERR_COUNT is reported. A draft that is no token is refused, rows that do not exist leave their sequence
 * without tokens (BS_DEV_ERR_BOUNDS). d_work: bs_draft_verify_work_bytes bytes, 16-byte aligned. */
uint64_t bs_draft_verify_work_bytes(uint32_t n_seqs, uint32_t vocab);
int bs_draft_verify(const bs_draft_batch *batch, void *d_work, uint64_t work_bytes, int32_t *d_status, void *stream);

#ifdef __cplusplus
}
#endif

#endif
