/*
 * trianglemix_pages.h -- C ABI of the paged serving operators of
 * libtrianglemix.so: key bounds of pages, page selection, attention over
 * selected pages, attention over draft trees.  Status codes, error text and
 * calling rules are those of trianglemix.h: every check runs on the host
 * before any HIP call; a call enqueues its kernels on `stream` and returns; it
 * allocates nothing, synchronises nothing and reads no device memory on the
 * host.  Lengths, tables, selections and masks live on the device and may
 * change between replays of a captured call.
 *
 * Common layout.  Heads of 128 dims, pages of 128 tokens, bf16 or fp16:
 *   caches       [num_pages, 128, kv_heads, 128], page strides in elements
 *                (the [128, kv_heads, 128] part contiguous, strides multiples of 8)
 *   block_table  [batch, table_cols] int32, logical page -> page of the cache,
 *                row stride in elements.  An entry that is no page of the cache
 *                (negative, or >= num_pages) is a page without keys.
 *   query, out   [batch * rows, heads, 128]; request b's rows are the last
 *                `rows` tokens of its first seq_lens[b], row t at position p =
 *                seq_lens[b] - rows + t.  A negative position is no row: it is
 *                neither read into a selection nor written.  query has a row
 *                stride in elements (a slice of a fused QKV buffer works); out
 *                is contiguous.
 * Query head h reads KV head h / (heads / kv_heads), any group of 1 to 32.
 * Tokens past table_cols * 128 have no page and no keys.
 * Limits: 1024 requests, 16384 table columns, 256 heads, 2^21 query rows,
 * 1024 pages per selection, 64 nodes per tree, 2^22 cache pages, and 2^30 pages
 * of attention work (pages per group, KV heads and groups of rows together).
 */
#ifndef TRIANGLEMIX_PAGES_H
#define TRIANGLEMIX_PAGES_H

#include <stdint.h>

#include "trianglemix.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TM_BF16 0
#define TM_FP16 1

/* Query rows that share one selection of pages. */
#define TM_SELECT_ROWS 32

/*
 * Elementwise smallest and largest key of every page that holds one of the
 * last num_tokens tokens of a request's first seq_lens[b], over the page's
 * tokens below seq_lens[b], into page_min / page_max [num_pages, kv_heads, 128]
 * (contiguous, the keys' type, exact).  A NaN among the keys makes both bounds
 * of its dim NaN.  Other pages' bounds are left as they were.  A length past
 * the table counts as the table's.  Call it after the tokens' K rows are in the
 * cache.  Requests may share pages that hold the same number of tokens for each
 * of them (a common prefix of full pages); with different lengths in a shared
 * page its bounds would be either's, in any mixture.
 */
int tm_update_page_bounds(const void* key_cache, int64_t key_page_stride, const int32_t* block_table,
                          int64_t table_stride, const int32_t* seq_lens, int64_t num_tokens, void* page_min,
                          void* page_max, int64_t batch, int64_t table_cols, int64_t num_pages, int64_t kv_heads,
                          int dtype, void* stream);

/*
 * The pages that each block of TM_SELECT_ROWS query rows should attend, per KV
 * head: out [batch, ceil(rows / 32), kv_heads, count] int32, logical pages in
 * ascending order, -1 behind them.  Of the pages up to the block's last row
 * that have keys: the first sink_pages, the recent_pages pages up to the one
 * of the block's first row and those after it (recent_pages 0: none), then
 * those with the largest
 *   score = max over the group's heads h of
 *           sum_d (qs_hd >= 0 ? qs_hd * max_d : qs_hd * min_d),
 * qs_h the sum of the block's query rows, summed in 64 bits; equal scores take
 * the lowest page, a score that is not a number ranks last.  Needs sink_pages +
 * recent_pages (+ 1 for more than one row) <= count.
 */
int tm_select_pages(const void* query, int64_t query_stride, const void* page_min, const void* page_max,
                    const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens, int32_t* out,
                    int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_cols,
                    int64_t num_pages, int64_t count, int64_t sink_pages, int64_t recent_pages, int dtype,
                    void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of that call, or -1 for what it refuses.  Any contents,
 * 16-byte aligned.  The call enqueues several launches that hand it on, so it
 * is one call's own until the last of them has run: no other call's launches,
 * from another thread on the same stream either, may come between them. */
int64_t tm_select_pages_workspace_size(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                       int64_t table_cols);

/*
 * Causal attention of each query row over the keys k <= p of the pages that
 * `pages` [batch, ceil(rows / 32), kv_heads, count] int32 lists for its block
 * and KV head.  The list is a set: any order, an entry twice counts once, an
 * entry that is no page up to the block's last row is ignored.
 *
 * Numerics, of this operator and of tm_tree_attention: scores, softmax
 * statistics and sums in fp32; the weights are rounded to the inputs' type for
 * their product with V (the sum that they are divided by takes them unrounded),
 * the result once more.  A row without keys gives zeros.  A key whose score is
 * -infinity counts as one that the row does not attend.  NaN, and infinities in V,
 * reach the rows that attend their key and no other; an infinity whose weight
 * rounds to zero may arrive as NaN.
 */
int tm_selected_page_attention(const void* query, int64_t query_stride, const void* key_cache,
                               int64_t key_page_stride, const void* value_cache, int64_t value_page_stride,
                               const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens,
                               const int32_t* pages, void* out, int64_t batch, int64_t rows, int64_t heads,
                               int64_t kv_heads, int64_t table_cols, int64_t num_pages, int64_t count, float scale,
                               int dtype, void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of that call, or -1 for what it refuses.  The workspace is
 * as that of tm_triangle_paged_sparse_attention: any contents, 16-byte
 * aligned, one per call in flight. */
int64_t tm_selected_page_attention_workspace_size(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                                  int64_t count);

/*
 * Attention of drafted tokens over the cache, one tree per request: request b
 * has the rows tree_offsets[b] .. tree_offsets[b + 1] - 1 of query, key, value
 * and out ([total_rows, heads or kv_heads, 128]; offsets int32 [batch + 1],
 * ascending), its nodes in any order.  Node i attends the first context_lens[b]
 * tokens of its request's cache and node j of the same tree where bit j of
 * tree_mask[tree_offsets[b] + i] (int64) is set; its own bit as the others.
 * The drafts' K and V rows are read from key / value (row strides in elements)
 * and are not in the cache.  A tree has at most 64 nodes; rows past a tree's
 * 64th node and rows of no request are left as they were.  A tree of one node
 * is a decoding step.  A node without keys gives zeros.
 */
int tm_tree_attention(const void* query, int64_t query_stride, const void* key, int64_t key_stride,
                      const void* value, int64_t value_stride, const void* key_cache, int64_t key_page_stride,
                      const void* value_cache, int64_t value_page_stride, const int32_t* block_table,
                      int64_t table_stride, const int32_t* context_lens, const int32_t* tree_offsets,
                      const int64_t* tree_mask, void* out, int64_t total_rows, int64_t batch, int64_t heads,
                      int64_t kv_heads, int64_t table_cols, int64_t num_pages, float scale, int dtype,
                      void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of that call, or -1 for what it refuses. */
int64_t tm_tree_attention_workspace_size(int64_t total_rows, int64_t batch, int64_t heads, int64_t kv_heads,
                                         int64_t table_cols);

#ifdef __cplusplus
}
#endif

#endif /* TRIANGLEMIX_PAGES_H */
