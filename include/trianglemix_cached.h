/*
 * trianglemix_cached.h -- C ABI of the cached-attention operators of
 * libtrianglemix.so: the position rotation of query and key rows, the rotated
 * write into a paged cache of 8-bit or 16-bit numbers, and attention over it.
 * Status codes, error text and calling rules are those of trianglemix.h, the
 * common layout and limits those of trianglemix_pages.h: every check runs on
 * the host before any HIP call; a call enqueues its kernels on `stream` and
 * returns; it allocates nothing, synchronises nothing and reads no device
 * memory on the host.  Positions, slots, lengths, tables and scales live on the
 * device and may change between replays of a captured call.
 *
 * Caches are [num_pages, 128, kv_heads, 128] as there, of the rows' own type
 * (cache_dtype TM_BF16 or TM_FP16, equal to dtype) or of e4m3 numbers (TM_E4M3:
 * 4 exponent bits of bias 7, 3 mantissa bits, largest 448, no infinities).  A
 * number of an e4m3 cache stands for itself times its KV head's scale,
 * key_scale / value_scale [kv_heads] fp32 (null for 16-bit caches): positive,
 * from 2^-126 to 2^126; others are not looked for and give numbers that mean
 * nothing.  Page strides are in numbers, of 16 bytes in multiples.  Of the
 * library's operators these alone read or write e4m3 caches; those of the other
 * headers take caches of 16 bits.
 */
#ifndef TRIANGLEMIX_CACHED_H
#define TRIANGLEMIX_CACHED_H

#include <stdint.h>

#include "trianglemix_pages.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TM_E4M3 2

/*
 * Rows of x [rows, heads, 128] rotated by their positions into out: for each
 * pair i < rotary_dim / 2 of a head's first rotary_dim dims,
 *   out_a = m (x_a cos(p f_i) - x_b sin(p f_i))
 *   out_b = m (x_b cos(p f_i) + x_a sin(p f_i))
 * with (a, b) = (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with `interleaved`,
 * p = positions[row] (int64), f = frequencies [rotary_dim / 2] fp64 (radians a
 * position) and m = magnitude.  The other dims are copied bit by bit.
 * rotary_dim is a multiple of 16 up to 128.  A negative position is no row: its
 * out is left as it was.  x and out have row strides in elements; out may be x
 * itself (the same pointer and stride), and must not overlap it otherwise.
 *
 * Numerics, of this operator and of tm_rotate_and_cache: the angle is reduced to
 * a turn in 64 bits (positions up to 2^30 and more), sine, cosine and products
 * are in 32, the result is rounded once.
 */
int tm_rotate_positions(const void* x, int64_t x_stride, const int64_t* positions, const double* frequencies,
                        void* out, int64_t out_stride, int64_t rows, int64_t heads, int64_t rotary_dim,
                        int interleaved, float magnitude, int dtype, void* stream);

/*
 * A step's projection output into the cache: row r's query heads rotated as
 * above into query_out, its keys rotated into slot slot_mapping[r] (int64: page
 * slot / 128, offset slot % 128) of key_cache, its values as they are into the
 * same slot of value_cache.  An e4m3 cache takes the nearest number (ties to
 * even) of the fp32 quotient by the head's scale, +-448 for what is larger, NaN
 * for NaN.  A row with a negative position is none and leaves everything as it
 * was; one whose slot is negative or past the cache is not stored, its query is
 * rotated all the same.  Rows that name one slot twice leave either's numbers,
 * in any mixture.  query_out may be query itself; views of one buffer whose rows
 * lie side by side (a fused QKV projection) do not overlap.
 */
int tm_rotate_and_cache(const void* query, int64_t query_stride, const void* key, int64_t key_stride,
                        const void* value, int64_t value_stride, const int64_t* positions,
                        const int64_t* slot_mapping, const double* frequencies, void* query_out,
                        int64_t query_out_stride, void* key_cache, int64_t key_page_stride, void* value_cache,
                        int64_t value_page_stride, const float* key_scale, const float* value_scale, int64_t rows,
                        int64_t heads, int64_t kv_heads, int64_t num_pages, int64_t rotary_dim, int interleaved,
                        float magnitude, int dtype, int cache_dtype, void* stream);

/*
 * Causal attention of the last `rows` tokens of each request over its pages:
 * the row at position p attends the keys k <= p, with window >= 0 only those
 * with k >= p - window or k < sinks.  window -1: all keys (sinks must be 0).
 * The step's own keys are in the cache.  Single tokens (rows 1), a few drafted
 * ones, or a whole chunk.  scale, times key_scale and log2(e), has to be a finite
 * number.
 *
 * The launch is planned for requests as long as their table is wide, and lengths
 * are found on the device: any length gives its result in any table, a short chunk
 * its best time in a table not much wider than the request.  A chunk of one request
 * in bf16, 32 heads over 8, all keys, over a contiguous 16-bit cache, is the work of
 * tm_dense_paged_causal_attention too: where its length is known on the host, that
 * call takes less time (512 rows of 8192 tokens 65 us, this one 81; 2048 of 32749 883
 * and 1013).
 *
 * A call may read 2^30 tiles of 32 keys, counted at the table's full width (the
 * window's, where there is one) for each request, each KV head (KV heads that a
 * workgroup has together count once) and, in chunks, each of their parts.  Keys
 * of pages that the cache does not have, and keys past the table, are attended
 * by no row.  Rows before a request's first token are none: their out is left as
 * it was.
 *
 * Numerics: scores, softmax statistics and sums in fp32.  The weights are rounded
 * to the cache's type for their product with V (fp16 over an e4m3 cache, whose
 * numbers are exact in it); the sum that they are divided by takes them
 * unrounded; the result is rounded once.  A row without keys gives zeros.  A key
 * whose score is -infinity has the weight zero.  NaN in keys, and NaN and
 * infinities in V, reach the rows that attend their key and no other, whatever
 * the key's weight; an infinity may arrive as NaN where that weight rounds to
 * zero or other infinities meet it.
 */
int tm_cached_attention(const void* query, int64_t query_stride, const void* key_cache, int64_t key_page_stride,
                        const void* value_cache, int64_t value_page_stride, const float* key_scale,
                        const float* value_scale, const int32_t* block_table, int64_t table_stride,
                        const int32_t* seq_lens, void* out, int64_t batch, int64_t rows, int64_t heads,
                        int64_t kv_heads, int64_t table_cols, int64_t num_pages, int64_t window, int64_t sinks,
                        float scale, int dtype, int cache_dtype, void* workspace, int64_t workspace_bytes,
                        void* stream);

/* Workspace bytes of that call over a cache of either type, or -1 for what it
 * refuses over both.  The workspace is
 * as that of tm_triangle_paged_sparse_attention: any contents, 16-byte
 * aligned, one per call in flight.  At most 64 MiB + 64 KiB. */
int64_t tm_cached_attention_workspace_size(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                           int64_t table_cols, int64_t window, int64_t sinks);

#ifdef __cplusplus
}
#endif

#endif /* TRIANGLEMIX_CACHED_H */
