/*
 * paged_ops.h — operators over a paged KV cache (B200).
 *
 * The reference moves and scores blocks of a paged cache but leaves writing
 * new tokens into it and attending over it to its callers.  These calls do
 * both on the pages where they lie, and give the block scores without an
 * attention map in memory:
 *
 *   orchkv_paged_append      norm of each head (optional), position rotation,
 *                            K and V into the pages, rotated Q out
 *   orchkv_paged_attend      attention of new tokens over the pages
 *   orchkv_paged_block_mass  attention mass of every block, what
 *                            tm_report_attn_batch_dev takes
 *
 * They keep no state, allocate nothing and run on the stream they are given
 * (any stream of the current device; capturable into a CUDA graph; lengths
 * and tables are read on the device, so a replayed graph follows them).
 * Every pointer is device memory.  Return codes are those of kv_types.h;
 * arguments are checked before anything is launched.
 */
#ifndef ORCHKV_PAGED_OPS_H
#define ORCHKV_PAGED_OPS_H

#include "orchkv_api.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The pages.  Element (page p, KV head h, token t, d) of K is at
 * k[p * page_stride + h * head_stride + t * token_stride + d], strides in
 * elements and not negative, V alike.  The data plane's slabs are pages of one head: k =
 * orchkv_gpu_pool_base(), v = k + half a slab, head_stride 0, page_stride
 * one slab.  k, v and every stride must be multiples of 16 bytes; d_head a
 * multiple of 16 bytes, at most 256 elements. */
typedef struct orchkv_pages {
    void    *k, *v;
    int64_t  page_stride, head_stride, token_stride;
    uint32_t n_pages;
    uint32_t page_tokens;
    uint32_t n_kv_heads;
    uint32_t d_head;
    int      dtype;               /* DTYPE_FP16, DTYPE_BF16 or DTYPE_FP32 */
} orchkv_pages_t;

/* One call's sequences.  Sequence i has its new tokens in rows
 * [starts[i], starts[i+1]) of the call's row tensors; they are the last of
 * its lens[i] tokens.  Token t of its KV head h lies in page
 * table[i * table_seq_stride + h * table_head_stride + t / page_tokens];
 * entries outside [0, n_pages) name no page.  starts must not decrease; rows
 * from starts[n_seqs] on belong to no sequence and are left alone.  max_new
 * is an upper bound of one sequence's new tokens (n_rows if unknown); the rows
 * of a sequence that has more may not be computed. */
typedef struct orchkv_batch {
    const int32_t *table;
    int64_t  table_seq_stride, table_head_stride;   /* head stride 0: one table for all heads */
    uint32_t table_width;
    uint32_t n_seqs;
    const int32_t *lens;
    const int32_t *starts;
    uint32_t n_rows;
    uint32_t max_new;
} orchkv_batch_t;

/* Row tensors: row r of head h at p[r * row_stride + h * head_stride], d_head
 * elements of the pages' dtype; pointer and strides multiples of 16 bytes. */
typedef struct orchkv_rows {
    void    *p;
    int64_t  row_stride, head_stride;
} orchkv_rows_t;

/* Position rotation: pair p < rot_dim/2 turns by turns[p] * position full
 * turns (device doubles; inv_freq / 2 pi).  Pairs are elements (p, p +
 * rot_dim/2), or (2p, 2p+1) when interleaved; elements from rot_dim on stay.
 * Both results are scaled by `scale`.  rot_dim 0: no rotation. */
typedef struct orchkv_append_args {
    orchkv_rows_t  q, q_out;      /* n_q_heads heads; n_q_heads 0: no queries */
    orchkv_rows_t  k, v;          /* n_kv_heads heads */
    uint32_t       n_q_heads;
    uint32_t       rot_dim;
    int            interleaved;
    float          scale;
    const double  *turns;
    const void    *positions;     /* per row; NULL: the token's place in its sequence */
    int            positions_64;  /* positions are int64 (else int32) */
    const void    *q_norm, *k_norm; /* [d_head] of the pages' dtype, or NULL: no norm */
    float          eps;
} orchkv_append_args_t;

/* x of a q or k head: y = x / sqrt(mean(x^2) + eps) * norm, if a norm is
 * given; y rotated, in fp32 and rounded once; k and v into the pages, q to
 * q_out (which may be q itself; else it must not overlap q, and never k, v or
 * itself).  Tokens whose table entry names no page are not
 * written (their q still is).  Every place of the pages must have memory of its
 * own (no zero stride over several pages, tokens or heads).  Asynchronous. */
int orchkv_paged_append(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                        const orchkv_append_args_t *args, void *stream);

typedef struct orchkv_attend_args {
    orchkv_rows_t  q, out;        /* n_q_heads heads */
    float         *lse;           /* [n_rows][n_q_heads], or NULL */
    uint32_t       n_q_heads;     /* a multiple of n_kv_heads */
    float          scale;
    uint32_t       window;        /* 0: all earlier tokens; else the last `window`, itself included */
} orchkv_attend_args_t;

/* out[r, h] = sum_t softmax_t(scale * q[r, h] . K[t]) V[t] over the tokens t
 * of r's sequence up to r's own place that lie in a page (and in the
 * window), KV head h / (n_q_heads / n_kv_heads); lse[r, h] = the logarithm of
 * the softmax's denominator.  A row with no such token gets 0 and -infinity,
 * and so does one whose scores are all -infinity.  For the second product the
 * weights are rounded to the pages' type (half a step each; fp16 ones are held
 * from 2^-25 of a row's largest up, and smaller ones to 2^-36 of it).
 * What lies in places that a row does not attend to does not reach it, be it
 * infinite or NaN; an infinite or NaN value reaches every row that does, as
 * such or as NaN.
 * out must not overlap q or itself.
 * workspace: orchkv_paged_attend_workspace() bytes of device memory, 256-byte
 * aligned, of this call alone until it has run.  Asynchronous. */
size_t orchkv_paged_attend_workspace(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                                     const orchkv_attend_args_t *args);
int orchkv_paged_attend(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                        const orchkv_attend_args_t *args, void *workspace, size_t bytes,
                        void *stream);

typedef struct orchkv_mass_args {
    orchkv_rows_t  q;
    const float   *lse;           /* [n_rows][n_q_heads], as orchkv_paged_attend gives it */
    float         *mass;          /* [n_seqs][n_kv_heads][table_width] */
    uint32_t       n_q_heads;
    float          scale;
    uint32_t       window;
} orchkv_mass_args_t;

/* mass[i, g, b] = sum over sequence i's rows r, the query heads h of KV head
 * g and the tokens t of block b of exp(scale * q[r, h] . K[t] - lse[r, h]),
 * the probability orchkv_paged_attend gave t: what tm_report_attn_probs sums
 * out of a stored map.  Blocks that hold no attended token get 0.  Sums run
 * in one fixed order.  pages->v is not read; mass must not overlap q or lse.  workspace as for
 * orchkv_paged_attend (NULL where the size is 0).  Asynchronous. */
size_t orchkv_paged_block_mass_workspace(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                                         const orchkv_mass_args_t *args);
int orchkv_paged_block_mass(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                            const orchkv_mass_args_t *args, void *workspace, size_t bytes, void *stream);

/* The data plane's GPU pool as pages of one head each, for requests of
 * n_kv_heads KV heads. */
int orchkv_pool_pages(uint32_t n_kv_heads, orchkv_pages_t *out);

/* The tables of these operators for one layer of the given requests (which
 * all have n_kv_heads KV heads and the same n_layers), device memory: table [n][n_kv_heads]
 * [ceil(row_len / tokens_per_block)] the GPU slab of each block, -1 where a
 * block does not exist or lies on another tier; lens [n] (may be NULL) the
 * tokens held.  New tokens get their blocks first: orchkv_append_token_batch
 * (one token, every layer) and orchkv_prefill (one layer) with NULL data
 * allocate and count them, orchkv_paged_append then writes them.
 * Runs on the data plane's stream: asynchronous while the requests are those of
 * the call before, behind a synchronisation of the stream when they are not. */
int orchkv_slab_table(kv_request_ctx_t *const *ctxs, uint32_t n, uint32_t layer_id, uint32_t n_kv_heads,
                      uint32_t row_len, int32_t *table, int32_t *lens);

/* ORCHKV_ERR_CUDA once a wait inside one of these kernels has run out (2 s;
 * its call's results are then not complete), ORCHKV_OK otherwise.
 * Synchronous. */
int orchkv_paged_status(void);

#ifdef __cplusplus
}
#endif
#endif /* ORCHKV_PAGED_OPS_H */
