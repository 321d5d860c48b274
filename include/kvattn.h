/*
 * Attention over the pages of a KV cache, for the tokens that a step feeds:
 * one token per sequence (decoding), a chain of them (drafted in a row, or a
 * chunk of a prompt), or a tree of drafted tokens.
 *
 * CrossCache leaves attention to the engine; this reads the paged geometries
 * that kvcopy.h moves (token-major, head-major, K and V side by side), so an
 * engine built on the library's cache needs no re-layout.
 *
 * Sequence b feeds the nodes q_offsets[b] .. q_offsets[b + 1) of the packed
 * queries, T of them; r = rows[b] (b without rows) is its row of the table.
 * The row holds lens[r] tokens, the fed ones last and in order, so that node j
 * stands at position lens[r] - T + j and its K and V have been written there.
 * With s = scale * k_scale * q . k, node j of head h computes
 *
 *   out = v_scale * sum_p softmax_p(s) V[p],   lse = log(sum_p exp(s_p))
 *
 * over the positions that it sees: every p < lens[r] - T, itself, and its
 * ancestors among the nodes.  K/V head h / (num_heads / num_kv_heads) serves
 * query head h.
 *
 * parents: [total_q] or NULL.  parents[q_offsets[b] + j] is the node of the
 * same sequence that node j follows: -1 .. j - 1, -1 for the last token before
 * the nodes.  -2 marks a padding node: it sees nothing (out 0, lse -inf), and
 * nothing sees it; its K and V may be anything.  NULL is a chain, parent j - 1.
 * A sequence without nodes is skipped, whatever its row.  Rows of out and lse
 * that no sequence covers are left as they were.  A row that sees nothing, or
 * only scores of -inf, is 0 with lse -inf.
 */
#ifndef __KVATTN_H__
#define __KVATTN_H__

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* bits the kernels OR into *error; all rows that are not named are right */
#define KVATTN_ERR_PAGE    0x1   /* a page id outside [0, num_pages); it counts as zeros */
#define KVATTN_ERR_SEQ     0x2   /* a row or length that fits neither table nor nodes: the sequence's rows are
                                  * 0 / -inf; or offsets out of order or past total_q: the sequence is skipped
                                  * (the results of queries that two others then both cover are unspecified) */
#define KVATTN_ERR_PARENT  0x4   /* a parent outside [-2, j - 1]: the node is taken for a padding node */
#define KVATTN_ERR_TIMEOUT 0x8   /* a wait inside the kernel ran out, after about a second: the results are void */

#define KVATTN_BF16 0
#define KVATTN_FP16 1
#define KVATTN_E4M3 2            /* caches only */

#define KVATTN_MAX_HEAD_DIM 256
#define KVATTN_MAX_SEQS     65536
#define KVATTN_MAX_QUERIES  (1u << 30)   /* total_q * num_heads */

struct kv_attn_desc {
    const void *q;               /* [total_q][num_heads][head_dim], see the strides */
    void *out;                   /* like q, same type */
    float *lse;                  /* [total_q][num_heads] or NULL */
    const void *k, *v;           /* plane bases of one layer, 16-byte aligned */
    const int32_t *table;        /* page ids, as in kvpage.h */
    const int32_t *lens;
    const int32_t *rows;         /* [num_seqs] or NULL */
    const int32_t *q_offsets;    /* [num_seqs + 1] */
    const int32_t *parents;
    int32_t *error;
    void *workspace;             /* kv_attn_workspace_bytes(), 256-byte aligned; nothing is kept in it between calls */
    uint64_t workspace_bytes;
    uint64_t block_stride;       /* bytes from page to page, 0 = block_size * num_kv_heads * head_dim * element */
    int64_t table_stride;
    int64_t q_stride, q_head_stride;      /* in elements, multiples of 8 above 0; head_dim is contiguous */
    int64_t out_stride, out_head_stride;
    uint32_t width;              /* entries of a table row */
    uint32_t num_rows;           /* rows of the table */
    uint32_t num_seqs;
    uint32_t total_q;
    uint32_t num_pages;
    uint32_t block_size;
    uint32_t num_heads;          /* at most 128 per K/V head */
    uint32_t num_kv_heads;
    uint32_t head_dim;           /* a multiple of 16, <= KVATTN_MAX_HEAD_DIM */
    uint32_t head_major;         /* pages are [kv heads][block_size][head_dim] */
    int32_t q_type;              /* KVATTN_BF16 or KVATTN_FP16 */
    int32_t kv_type;             /* q_type or KVATTN_E4M3 */
    float scale, k_scale, v_scale;        /* scale and k_scale above 0 */
    int32_t device;
};

/* Bytes of workspace that a call of `desc` needs (its pointers are not
 * looked at), or a negative errno. */
int64_t kv_attn_workspace_bytes(const struct kv_attn_desc *desc);

/* Asynchronous on `stream`, allocates nothing, may be captured.  Returns 0,
 * -EINVAL for a malformed descriptor, -E2BIG past KVATTN_MAX_SEQS or
 * KVATTN_MAX_QUERIES, or -EIO when the launch failed. */
int kv_attn_launch(const struct kv_attn_desc *desc, void *stream);

/* For tests of the failure detection: the same, but in the grid's first CTA
 * (where it has work) the first tile of V counts as never loaded.  The waits for
 * it run out after some 20 milliseconds, KVATTN_ERR_TIMEOUT is set, and what is
 * in flight settles before the CTA leaves.  The results are void. */
int kv_attn_launch_stalled(const struct kv_attn_desc *desc, void *stream);

#ifdef __cplusplus
}
#endif

#endif
