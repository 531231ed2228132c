/*
 * bigsmall_kv.h — C ABI of the paged 8-bit KV cache (libbigsmall_hip.so):
 * appending with the position rotation, attention over the cache, and reading
 * a sequence back in bf16. No reference counterpart: the reference stores K/V
 * entries (bigsmall/kv_cache_manager.py:22-91) and leaves attention to torch.
 *
 * As in bigsmall_hip.h: plain pointers and sizes, `stream` a hipStream_t as
 * void*, calls asynchronous on it, negative BS_ERR_* codes for what the host
 * can see, BS_DEV_ERR_BOUNDS OR-ed into *d_status (may be NULL) for page or
 * tail numbers, lengths or offsets in device memory that are out of range:
 * what they name is neither read nor written. No call allocates, synchronises
 * or keeps state; all may be captured into a graph.
 */
#ifndef BIGSMALL_KV_H
#define BIGSMALL_KV_H

#include <stdint.h>

#include "bigsmall_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define BS_KV_PAGE 64 /* tokens per page */
#define BS_KV_INT8 0
#define BS_KV_FP8 1 /* e4m3 (OCP, finite) */

/* One layer's storage, device memory, 16-byte aligned. A full page is held in
 * 8 bits with one scale per kv head for K and one for V; the tokens of a
 * sequence's unfinished page are held in bf16 in a tail, from which the page
 * is quantised once, when it is full. Value = code * scale. bs_kv_attend takes
 * v_scale as bs_kv_append leaves it, positive and between 2^-49 and 2^54 (a page
 * of zeros among them): under a v_scale of 0 a page's keys lose their weight. */
typedef struct {
    void *k;            /* [n_pages][n_kv_heads][64][head_dim] */
    void *v;            /* [n_pages][n_kv_heads][head_dim][64]: tokens innermost */
    float *k_scale;     /* [n_pages][n_kv_heads] */
    float *v_scale;
    uint16_t *k_tail;   /* [n_tails][n_kv_heads][64][head_dim], bf16 */
    uint16_t *v_tail;   /* [n_tails][n_kv_heads][head_dim][64], bf16 */
    uint32_t n_pages, n_tails, n_kv_heads;
    uint32_t head_dim;  /* 64, 80, 96, 128 or 256 */
    uint32_t kind;      /* BS_KV_INT8 or BS_KV_FP8 */
} bs_kv_pool;

/* One step over a batch of sequences, device memory. max_new and max_len are
 * the largest of their kind over the sequences; they choose launch shapes and
 * do not bound the work (a wrong value costs time, not results). Rows that no
 * sequence covers are not read, and their outputs are not defined. */
typedef struct {
    const int32_t *start; /* [n_seqs] tokens in the cache before the step */
    const int32_t *cu;    /* [n_seqs + 1] first new row of each sequence, ascending from 0 */
    const int32_t *table; /* [n_seqs][table_stride], the first table_cols page numbers of a row used */
    const int32_t *tails; /* [n_seqs][2] the tail before the step, the tail after it; where the step
                             completes a page they differ, else they may be one */
    uint32_t n_seqs, table_stride, table_cols;
    uint32_t n_rows;      /* new rows in all */
    uint32_t max_new, max_len;
} bs_kv_batch;

/* bf16 rows [n_rows][heads][head_dim]; strides in elements, multiples of 8,
 * the last dimension contiguous, bases 16-byte aligned. */
typedef struct {
    const uint16_t *q;  /* may be NULL: nothing to rotate */
    const uint16_t *k;
    const uint16_t *v;
    uint16_t *q_out;    /* [n_rows][n_q_heads][head_dim], contiguous; may be q itself if that is contiguous */
    const float *cos;   /* [n_pos][rot / 2]; NULL with rot 0 */
    const float *sin;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    uint32_t n_q_heads; /* a multiple of the pool's kv heads */
    uint32_t rot;       /* channels that turn, from the first on: a multiple of 8, at most head_dim; 0: none */
    uint32_t interleaved; /* pairs: 0 (i, i + rot/2), 1 (2i, 2i + 1) */
    uint32_t n_pos;     /* rows of cos and sin */
} bs_kv_rows;

/* Rotate q and k by their tokens' positions (f32, rounded to bf16), write k
 * and v into the cache: full pages as codes and scales, the rest into the
 * sequence's tail. For a page a = max |x| held to [2^-40, 2^60]; scale =
 * a * (1 / qmax), code = x * (qmax * (1 / a)) rounded to nearest even, qmax 127
 * or 448. A token with a non-finite rotated k or v in a head is poisoned
 * there: its k is stored as NaN, v's non-finite values as 0, so that exactly
 * the rows that see it become NaN (in a full page, the rows that see any
 * token of the page: its k scale is NaN). Running a step again gives the same
 * cache as long as tails[b] differ wherever a page is completed. */
int bs_kv_append(const bs_kv_pool *pool, const bs_kv_batch *batch, const bs_kv_rows *rows, int32_t *d_status,
                 void *stream);

typedef struct {
    const uint16_t *q;  /* bf16 rows as in bs_kv_rows, rotated */
    uint16_t *out;      /* [n_rows][n_q_heads][head_dim], contiguous */
    float *lse;         /* [n_rows][n_q_heads], natural log; may be NULL */
    const float *slopes;   /* [n_q_heads] distance bias; may be NULL */
    const int32_t *prefix; /* [n_seqs]; may be NULL */
    const int32_t *first;  /* [n_rows]; may be NULL */
    int64_t q_token, q_head;
    uint32_t n_q_heads;
    uint32_t window;    /* 0: none */
    float scale;        /* of q . k */
    float softcap;      /* 0: none; others are held to [2^-60, 2^60] */
} bs_kv_query;

/* Attention of each new row over its sequence's cache, the step's own tokens
 * included (append first). Score s = scale * q.k, then softcap * tanh(s /
 * softcap), then minus slope * |p - j|; key j is seen by the row at position p
 * if j <= p or j < prefix, and j >= first, and j > p - window. A row that sees
 * nothing gives 0 and lse -inf. Scores, softmax and sums are f32; the weights
 * are f16 in the product with V (over a tail two bf16 parts). d_work: bs_kv_attend_work_bytes bytes of
 * scratch, 16-byte aligned (0 bytes may be NULL). */
uint64_t bs_kv_attend_work_bytes(const bs_kv_pool *pool, const bs_kv_batch *batch, uint32_t n_q_heads);
int bs_kv_attend(const bs_kv_pool *pool, const bs_kv_batch *batch, const bs_kv_query *query, void *d_work,
                 uint64_t work_bytes, int32_t *d_status, void *stream);

/* One sequence's first n tokens as bf16 [n_kv_heads][n][head_dim]: d_pages its
 * page numbers (n_cols of them), d_tail its tail's number (read if n is no
 * multiple of 64). */
int bs_kv_read(const bs_kv_pool *pool, const int32_t *d_pages, uint32_t n_cols, const int32_t *d_tail, uint32_t n,
               uint16_t *d_k, uint16_t *d_v, int32_t *d_status, void *stream);

#ifdef __cplusplus
}
#endif

#endif
