// Internal interface of the paged serving operators (page bounds, page
// selection, attention over selected pages, attention over draft trees)
// between their host code and their kernels.
#ifndef TRIANGLEMIX_PAGES_INTERNAL_H
#define TRIANGLEMIX_PAGES_INTERNAL_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "trianglemix_kernel.h"

namespace tmx {

// Limits of these operators (the attention operators' head size and page size
// are those of trianglemix_kernel.h).
constexpr int kSelectRows = 32;       // query rows that share one selection
constexpr int kMaxGroup = 32;         // query heads per KV head
constexpr int kMaxBatch = 1024;       // requests of one call
constexpr int kMaxSelected = 1024;    // pages of one selection
constexpr int kMaxTableCols = 16384;  // logical pages of a request (2,097,152 tokens)
constexpr int kMaxUnits = 1 << 30;    // pages of 128 keys that a call may read, per KV head and group of rows
constexpr int kMaxTreeNodes = 64;     // one 64-bit mask word per node

struct BoundsParams {
  const uint16_t* key_cache;
  int64_t page_stride;  // elements
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* seq_lens;
  uint16_t* page_min;  // [num_pages, kv_heads, 128]
  uint16_t* page_max;
  int table_cols, batch, kv_heads, num_pages, num_tokens;
};
hipError_t launch_page_bounds(const BoundsParams& p, bool fp16, hipStream_t stream);

struct SelectParams {
  const uint16_t* query;  // [batch * rows, heads, 128]
  int64_t query_stride;   // elements
  const uint16_t* page_min;
  const uint16_t* page_max;
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* seq_lens;
  int32_t* out;     // [batch, blocks, kv_heads, count]
  double* pooled;    // [slab requests * slab blocks, heads, 128] (more than one row), or null
  uint64_t* scores;  // [slab requests * slab blocks, kv_heads, table_cols]
  int table_cols, batch, rows, blocks, heads, kv_heads, num_pages, count, sink_pages, recent_pages;
  // The slab of requests and row blocks of one launch: their scores fit the workspace.
  int request0, requests, block0, slab_blocks;
};
hipError_t launch_select_pages(const SelectParams& p, bool fp16, hipStream_t stream);

// Attention of groups of query rows over lists of pages (trianglemix_rows.hip).
struct RowsParams {
  const uint16_t* query;  // [total_rows, heads, 128]
  int64_t query_stride;   // elements
  const char* key_cache;
  const char* value_cache;
  int64_t key_page_stride;  // bytes
  int64_t value_page_stride;
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* lens;      // seq_lens, or the context lengths of trees
  const int32_t* selected;  // [batch, blocks, kv_heads, count]; null for trees
  const char* draft_key;    // [total_rows, kv_heads, 128], trees alone
  const char* draft_value;
  int64_t draft_key_stride;  // bytes
  int64_t draft_value_stride;
  const int32_t* tree_offsets;  // [batch + 1]
  const int64_t* tree_mask;     // [total_rows]
  uint16_t* out;                // [total_rows, heads, 128]
  unsigned long long* counters;
  float* partials;
  unsigned long long epoch;
  int table_cols, batch, heads, kv_heads, group, num_pages, total_rows;
  int rows, blocks, count;  // selected pages: rows per request, row blocks per request, pages per selection
  int workgroups;           // of the grid
  int total_units, per_run;  // selected pages: all units, and those of a workgroup
  float scale_log2;
};
// Rows of one workgroup: groups of up to 32 rows run in trianglemix_rows.hip,
// larger ones in trianglemix_blocks.hip, of more than 256 rows in several
// workgroups.  Measured: 24 pages for each of 64 requests' 4 rows a KV head
// 137 us with 16 rows, 152 with 256; a 28-row tree 9.4 with 32, 11.1 with 256;
// 32 trees of up to 128 rows over 8000 tokens 192 with 128, 208 with 256.
constexpr int kComputeUnits = 256;  // of an MI355X, in 8 XCDs
constexpr int kFewRows = 16, kMostStreamRows = 32, kHalfBlockRows = 128, kBlockRows = 256;
// A run of units leaves at most two partial records of this many bytes.
constexpr int64_t rows_partial_bytes(int rows) {
  return rows > kMostStreamRows ? kPartialBytes * (rows / 128) : int64_t(rows) * (kHeadDim + 2) * 4;
}
// Fewest units of a run where a group has `units`: a small group is not split,
// as its partials and their merge cost more than reading three pages one after the
// other (a 7-node tree behind 77 tokens: 9.5 us in one run, 11.0 in two; 64
// blocks of three pages each: 26.2 and 26.9); a run of the large shapes takes two.
__host__ __device__ constexpr int min_run_units(int units, int rows) {
  return units <= 3 ? (units < 1 ? 1 : units) : rows > kMostStreamRows ? 2 : 1;
}
hipError_t launch_rows_attention(const RowsParams& p, int shape_rows, bool fp16, hipStream_t stream);
hipError_t launch_blocks_attention(const RowsParams& p, int shape_rows, bool fp16, hipStream_t stream);

// From trianglemix_capi.cpp: the calling thread's last error text (returns
// status), and the arrival tag of a launch on this workspace.
int report(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
unsigned long long workspace_tag(const void* workspace);

}  // namespace tmx

#endif  // TRIANGLEMIX_PAGES_INTERNAL_H
