/*
 * Pages of a paged KV cache, owned and moved on the device: allocating and
 * freeing them (resize), sharing them between sequences (fork), copying them
 * (copy) and squeezing dropped tokens out of them (compact).
 *
 * CrossCache moves pages that an engine's own block manager owns
 * (src/cache/cache.c:345-425); it has no counterpart of these entry points.
 * They are for an engine that keeps its block tables on the GPU: the
 * operators between a load and a store, on the paged geometries of kvcopy.h.
 *
 * The state is five int32 device arrays and no host copy:
 *   table      [num_rows][table_stride] page ids; row r (a sequence) holds the
 *              pages table[r][0 .. ceil(lens[r] / block_size)); the entries
 *              behind them are left as they were
 *   lens       [num_rows] tokens of each row, 0 = an empty row
 *   refs       [num_pages] rows that hold the page, 0 = a free page
 *   free_list  [num_pages] a stack: the free pages are free_list[0 ..
 *              *free_count), the last one is taken first
 *   free_count [1]
 * The state's calls are made on one stream, or ordered by the caller; they
 * allocate nothing, do not synchronise, and may be captured into a graph.
 * Their results do not depend on the order in which threads run, but for the
 * place in the free list of a page that a call gives back too often
 * (KVPAGE_ERR_REFS).  What a call is given is read before the state is written:
 * it may be part of the state.
 *
 * The launch functions return 0, -EINVAL for a malformed argument, -E2BIG
 * past a limit below, -EIO when the launch failed.  What only the device can
 * see sets bits in *error and is left alone, the rest of the call is done:
 * rows with status KVPAGE_INVALID are as they were, and where a call does
 * anything else with what is wrong, it says so below.
 */
#ifndef __KVPAGE_H__
#define __KVPAGE_H__

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* bits the kernels OR into *error */
#define KVPAGE_ERR_PAGE   0x1   /* a page id outside [0, num_pages): in the arguments, a row or the free list */
#define KVPAGE_ERR_ROW    0x2   /* a row outside the table, named twice in a call, a length that does not fit it;
                                 * fork: a child that is not empty, or that is also a parent */
#define KVPAGE_ERR_REFS   0x4   /* a page given back by a row that no longer held it; compact: a token to be moved
                                 * into a page that another row holds too */
#define KVPAGE_ERR_KEEP   0x8   /* compact: kept tokens not strictly ascending within [start, length) */
#define KVPAGE_ERR_ALIGN  0x10  /* a null or misaligned layer base: copies leave that plane out, compact refuses its rows */

/* a row's result in status[] */
#define KVPAGE_OK         0
#define KVPAGE_NO_PAGES   1     /* not enough free pages: the row is as it was */
#define KVPAGE_INVALID    2     /* an error bit says why: the row is as it was */

#define KVPAGE_ANY_DEVICE -1

#define KVPAGE_MAX_CALL   4096  /* rows of one resize / fork / compact call */
#define KVPAGE_MAX_ROWS   65536 /* rows of a table */

struct kv_page_state {
    int32_t *table;
    int32_t *lens;
    int32_t *refs;
    int32_t *free_list;
    int32_t *free_count;
    int32_t *marks;          /* [num_pages] scratch: zeros before the first call, zeros after each call */
    int32_t *error;          /* [1], never cleared by the calls */
    int64_t table_stride;    /* entries from one row to the next */
    uint32_t width;          /* entries of a row, <= table_stride */
    uint32_t num_rows;
    uint32_t num_pages;
    uint32_t block_size;     /* tokens per page */
    int32_t device;
};

/* where the pages are: the geometry of kv_copy_desc */
struct kv_page_cache {
    const uint64_t *layer_k; /* device array [num_layers] of K plane bases */
    const uint64_t *layer_v; /* V plane bases, or NULL for a K-only cache */
    int32_t *error;
    uint64_t block_stride;   /* bytes from one page of a plane to the next, 0 = block_size * unit_bytes */
    uint32_t unit_bytes;     /* bytes per token per layer per K/V */
    uint32_t head_bytes;     /* > 0: head-major pages */
    uint32_t block_size;
    uint32_t num_layers;
    uint32_t num_pages;
    uint32_t base_align;     /* a power of two that divides every plane base; 0 = 16 */
    int32_t device;
};

/* The device whose memory ptr points to, KVPAGE_ANY_DEVICE for memory that all
 * devices reach (pinned or managed), -EINVAL for any other. */
int kv_page_device_of(const void *ptr);

/* Set row rows[i] to lens[i] tokens, i < n: pages are given back where that
 * takes fewer, and taken where it takes more (what they hold is not touched).
 * An id in the free list that is no page goes to the row whose turn it is as it
 * stands, with KVPAGE_ERR_PAGE set, and is nobody's again once it is given back.
 * First all rows that shrink give back their entries.  A page whose last
 * reference goes is pushed; where several rows drop it, its place in the
 * order is that of the last.  Then the rows that grow take pages, in the order
 * of the call: row i is served if the pages that it and the rows before it in
 * the call ask for are there (status KVPAGE_NO_PAGES otherwise).
 * lens[i] = 0 frees a row.  A row that now ends inside a page which another
 * row holds too is not to be appended to there.  status: [n] or NULL. */
int kv_page_resize_launch(const struct kv_page_state *state, const int32_t *rows, const int32_t *lens,
                          uint32_t n, int32_t *status, void *stream);

/* Copy page src[i] to page dst[i] in every layer, K and V; with tokens, only
 * its first tokens[i] tokens.  A destination is named once and is not a source
 * of another pair: otherwise what that page (and no other) holds afterwards is
 * unspecified. */
int kv_page_copy_launch(const struct kv_page_cache *cache, const int32_t *src, const int32_t *dst,
                        const int32_t *tokens, uint32_t n, void *stream);

/* Make the empty row children[i] a continuation of row parents[i], i < n:
 * it shares the parent's full pages and gets a copy of the tokens of a partly
 * filled last page, in a page of its own, so that both can be appended to.
 * Pages are taken in the order of the call as in resize.  A row may be the
 * parent of many.  A child whose parent holds an id that is no page, or whose
 * turn it is for one of the free list, stays empty (KVPAGE_INVALID; the latter
 * id is off the list).  pairs: scratch of 3 * n int32. */
int kv_page_fork_launch(const struct kv_page_cache *cache, const struct kv_page_state *state,
                        const int32_t *parents, const int32_t *children, uint32_t n, int32_t *pairs,
                        int32_t *status, void *stream);

/* Keep some of the tokens of row rows[i], i < n: tokens before start[i] stay,
 * token start[i] + j becomes the one at position keep[offsets[i] + j],
 * j < offsets[i + 1] - offsets[i], in every layer, K and V; the row's length
 * becomes start[i] + the number kept, and the pages behind it are given back
 * as by resize.  keep: num_keep positions, strictly ascending in
 * [start[i], lens[row]) for each row.  The pages written to must be held by
 * that row alone.  scratch: n int32. */
int kv_page_compact_launch(const struct kv_page_cache *cache, const struct kv_page_state *state,
                           const int32_t *rows, const int32_t *start, const int32_t *keep,
                           const int32_t *offsets, uint32_t num_keep, uint32_t n, int32_t *scratch,
                           int32_t *status, void *stream);

#ifdef __cplusplus
}
#endif

#endif
