// C ABI of the paged serving operators (include/trianglemix_pages.h): host
// checks and launch geometry.  Every check runs before any HIP call.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/trianglemix_pages.h"
#include "trianglemix_checks.h"
#include "trianglemix_pages.h"

static_assert(TM_SELECT_ROWS == tmx::kSelectRows, "the public block size is the kernels'");

namespace {

using namespace tmx;

// Scores are kept for slabs of requests and row blocks of at most this many
// bytes (one block of the most KV heads and table columns takes 33 MB).
constexpr int64_t kSlabBytes = int64_t(40) << 20;

struct Slab {
  int64_t requests, blocks, pooled_bytes, bytes;
};

Slab select_slab(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_cols) {
  const int64_t blocks = (rows + tmx::kSelectRows - 1) / tmx::kSelectRows;
  const int64_t pooled = rows > 1 ? heads * tmx::kHeadDim * 8 : 0;
  const int64_t each = pooled + kv_heads * table_cols * 8;
  Slab s;
  s.blocks = std::min(blocks, std::max<int64_t>(1, kSlabBytes / each));
  s.requests = s.blocks < blocks ? 1 : std::min(batch, std::max<int64_t>(1, kSlabBytes / (each * blocks)));
  s.pooled_bytes = s.requests * s.blocks * pooled;
  s.bytes = s.requests * s.blocks * each;
  return s;
}

int check_select(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_cols) {
  int st = check_batch(batch, rows, batch * std::max<int64_t>(rows, 0));
  if (st == TM_OK) st = check_heads(heads, kv_heads);
  if (st == TM_OK) st = check_table(table_cols, table_cols, batch);
  return st;
}

// Rows of the workgroup shape for groups of `rows` rows.
int shape_for(int64_t rows) {
  for (int shape : {tmx::kFewRows, tmx::kMostStreamRows, tmx::kHalfBlockRows}) {
    if (rows <= shape) return shape;
  }
  return tmx::kBlockRows;
}

struct RowsPlan {
  int shape, workgroups;
  int64_t units, per_run, workspace_bytes;
};

// As many workgroups as `slots`, what the GPU holds at once, fewer when there are not as
// many units (pages of groups of rows); a multiple of the 8 XCDs.
RowsPlan rows_plan(int shape, int64_t units, int64_t min_units, int64_t slots = tmx::kComputeUnits) {
  RowsPlan r;
  r.shape = shape;
  r.units = units;
  r.workgroups = (int)((std::min<int64_t>(slots, (units + min_units - 1) / min_units) + 7) / 8 * 8);
  r.per_run = std::max(min_units, (units + r.workgroups - 1) / r.workgroups);
  r.workspace_bytes = tmx::kCounterBytes + 2 * r.workgroups * tmx::rows_partial_bytes(r.shape);
  return r;
}

int launch_attention(const tmx::RowsParams& p, const RowsPlan& plan, int dtype, void* stream) {
  const bool fp16 = dtype == TM_FP16;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return launched(plan.shape > tmx::kMostStreamRows ? tmx::launch_blocks_attention(p, plan.shape, fp16, s)
                                                     : tmx::launch_rows_attention(p, plan.shape, fp16, s));
}

int check_selected(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t count) {
  int st = check_batch(batch, rows, batch * std::max<int64_t>(rows, 0));
  if (st == TM_OK) st = check_heads(heads, kv_heads);
  if (st != TM_OK) return st;
  if (count <= 0) return report(TM_ERR_INVALID_ARGUMENT, "pages must list at least one page per block and KV head");
  if (count > tmx::kMaxSelected) {
    return report(TM_ERR_UNSUPPORTED, "%lld pages per selection; the limit is %d", (long long)count, tmx::kMaxSelected);
  }
  return TM_OK;
}

RowsPlan selected_plan(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t count) {
  const int64_t group_rows = std::min<int64_t>(rows, tmx::kSelectRows) * (heads / kv_heads);
  const int shape = shape_for(group_rows);
  const int64_t blocks = (rows + tmx::kSelectRows - 1) / tmx::kSelectRows;
  const int64_t groups = batch * blocks * kv_heads * ((group_rows + shape - 1) / shape);
  // Groups of up to 128 rows run in workgroups of eight waves, one a CU.  With two
  // groups a CU and more, in workgroups of four, two a CU: one starts its next
  // group beside the other's tiles.  Eight | four waves: 512 groups of 32 pages
  // of 131072 tokens 182 | 170 us, of 8 pages of 8192 tokens 52 | 45; 256 groups
  // of 32 pages 79 | 83, of 64 pages, each read once, 200 | 224; 128 groups of 16
  // pages 34 | 38.  (Lists of 4 to 8 pages lose 0.5 to 1 us of 20 to 25 by the key
  // parts' join against eight row parts, four of them empty.)
  const bool two = shape == tmx::kHalfBlockRows && groups >= 2 * tmx::kComputeUnits;
  return rows_plan(shape, groups * count, tmx::min_run_units((int)count, shape), (two ? 2 : 1) * tmx::kComputeUnits);
}

int check_tree(int64_t total_rows, int64_t batch, int64_t heads, int64_t kv_heads, int64_t table_cols) {
  int st = check_batch(batch, 0, total_rows);
  if (st == TM_OK) st = check_heads(heads, kv_heads);
  if (st == TM_OK) st = check_table(table_cols, table_cols, batch);
  return st;
}

// The shape holds the trees that the batch's average lets expect: equal ones
// where the rows divide evenly, else up to a quarter more than it.  A larger tree
// takes several row parts, each reading the request's K/V again: 32 trees of 5 to
// 10 nodes (up to 40 rows a KV head) take 146 us in the shape for 128 rows, 151 in
// parts of 32; of 4 to 8 nodes 207 and, in one part each, 194.
// A ragged batch whose rows happen to divide evenly is taken for one of equal
// trees: 32 of 4 to 12 nodes, 256 in all, 288 us, with 257 in all 199 (32 of 8: 192).
RowsPlan tree_plan(int64_t total_rows, int64_t batch, int64_t heads, int64_t kv_heads, int64_t table_cols) {
  const int64_t group = heads / kv_heads;
  const int64_t expected = total_rows % batch == 0 ? total_rows / batch : (5 * total_rows + 4 * batch - 1) / (4 * batch);
  const int shape = shape_for(std::min<int64_t>(expected, tmx::kMaxTreeNodes) * group);
  const int64_t groups = kv_heads * (batch + total_rows * group / shape);
  return rows_plan(shape, groups * (table_cols + 1), 1);  // the device deals the units that there are
}

}  // namespace

extern "C" {

int tm_update_page_bounds(const void* key_cache, int64_t key_page_stride, const int32_t* block_table,
                          int64_t table_stride, const int32_t* seq_lens, int64_t num_tokens, void* page_min,
                          void* page_max, int64_t batch, int64_t table_cols, int64_t num_pages, int64_t kv_heads,
                          int dtype, void* stream) {
  int st = check_dtype(dtype);
  if (st == TM_OK) st = check_batch(batch, num_tokens, 0);
  if (st == TM_OK) st = check_heads(kv_heads, kv_heads);
  if (st == TM_OK) st = check_table(table_cols, table_stride, batch);
  if (st == TM_OK) st = check_cache(num_pages, key_page_stride, kv_heads, "key_cache");
  if (st != TM_OK || batch == 0 || num_tokens == 0) return st;
  st = check_aligned({key_cache, page_min, page_max});
  if (st == TM_OK) st = check_element(block_table, 4);
  if (st == TM_OK) st = check_element(seq_lens, 4);
  if (st != TM_OK) return st;
  const int64_t bounds = num_pages * kv_heads * kHeadBytes;
  const Range written[] = {{page_min, bounds, "page_min"}, {page_max, bounds, "page_max"}};
  const Range read[] = {{key_cache, cache_bytes(num_pages, key_page_stride, kv_heads), "key_cache"},
                        {block_table, table_bytes(batch, table_stride, table_cols), "block_table"},
                        {seq_lens, batch * 4, "seq_lens"}};
  st = check_overlap(written, read);
  if (st != TM_OK) return st;
  tmx::BoundsParams p{};
  p.key_cache = static_cast<const uint16_t*>(key_cache);
  p.page_stride = key_page_stride;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.seq_lens = seq_lens;
  p.page_min = static_cast<uint16_t*>(page_min);
  p.page_max = static_cast<uint16_t*>(page_max);
  p.table_cols = (int)table_cols;
  p.batch = (int)batch;
  p.kv_heads = (int)kv_heads;
  p.num_pages = (int)num_pages;
  p.num_tokens = (int)num_tokens;
  return launched(tmx::launch_page_bounds(p, dtype == TM_FP16, static_cast<hipStream_t>(stream)));
}

int64_t tm_select_pages_workspace_size(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                       int64_t table_cols) {
  report(TM_OK, "%s", "");
  if (check_select(batch, rows, heads, kv_heads, table_cols) != TM_OK) return -1;
  return batch == 0 || rows == 0 ? 0 : select_slab(batch, rows, heads, kv_heads, table_cols).bytes;
}

int tm_select_pages(const void* query, int64_t query_stride, const void* page_min, const void* page_max,
                    const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens, int32_t* out,
                    int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_cols,
                    int64_t num_pages, int64_t count, int64_t sink_pages, int64_t recent_pages, int dtype,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  int st = check_dtype(dtype);
  if (st == TM_OK) st = check_select(batch, rows, heads, kv_heads, table_cols);
  if (st == TM_OK) st = check_selected(batch, rows, heads, kv_heads, count);
  if (st == TM_OK) st = check_table(table_cols, table_stride, batch);
  if (st == TM_OK) st = check_cache(num_pages, tmx::kPageSize * kv_heads * tmx::kHeadDim, kv_heads, "the cache");
  if (st == TM_OK) st = check_stride(query_stride, heads * tmx::kHeadDim, batch * rows, "query");
  if (st != TM_OK) return st;
  if (sink_pages < 0 || recent_pages < 0 || sink_pages > count || recent_pages > count ||
      sink_pages + recent_pages + (rows > 1 ? 1 : 0) > count) {
    return report(TM_ERR_INVALID_ARGUMENT,
                  "sink_pages and recent_pages must not be negative and leave count at least the pages that they take");
  }
  if (batch == 0 || rows == 0) return TM_OK;
  st = check_aligned({query, page_min, page_max});
  if (st == TM_OK) st = check_element(block_table, 4);
  if (st == TM_OK) st = check_element(seq_lens, 4);
  if (st == TM_OK) st = check_element(out, 4);
  if (st != TM_OK) return st;
  const Slab slab = select_slab(batch, rows, heads, kv_heads, table_cols);
  st = check_workspace(workspace, workspace_bytes, slab.bytes);
  if (st != TM_OK) return st;
  const int64_t blocks = (rows + tmx::kSelectRows - 1) / tmx::kSelectRows;
  const int64_t bounds = num_pages * kv_heads * kHeadBytes;
  const Range written[] = {{out, batch * blocks * kv_heads * count * 4, "out"}, {workspace, slab.bytes, "workspace"}};
  const Range read[] = {{query, rows_bytes(batch * rows, query_stride, heads * tmx::kHeadDim), "query"},
                        {page_min, bounds, "page_min"},
                        {page_max, bounds, "page_max"},
                        {block_table, table_bytes(batch, table_stride, table_cols), "block_table"},
                        {seq_lens, batch * 4, "seq_lens"}};
  st = check_overlap(written, read);
  if (st != TM_OK) return st;
  tmx::SelectParams p{};
  p.query = static_cast<const uint16_t*>(query);
  p.query_stride = query_stride;
  p.page_min = static_cast<const uint16_t*>(page_min);
  p.page_max = static_cast<const uint16_t*>(page_max);
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.seq_lens = seq_lens;
  p.out = out;
  p.pooled = slab.pooled_bytes > 0 ? static_cast<double*>(workspace) : nullptr;
  p.scores = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + slab.pooled_bytes);
  p.table_cols = (int)table_cols;
  p.batch = (int)batch;
  p.rows = (int)rows;
  p.blocks = (int)blocks;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.num_pages = (int)num_pages;
  p.count = (int)count;
  p.sink_pages = (int)sink_pages;
  p.recent_pages = (int)recent_pages;
  for (int64_t b = 0; b < batch; b += slab.requests) {
    for (int64_t k = 0; k < blocks; k += slab.blocks) {
      p.request0 = (int)b;
      p.requests = (int)std::min(slab.requests, batch - b);
      p.block0 = (int)k;
      p.slab_blocks = (int)std::min(slab.blocks, blocks - k);
      st = launched(tmx::launch_select_pages(p, dtype == TM_FP16, static_cast<hipStream_t>(stream)));
      if (st != TM_OK) return st;
    }
  }
  return TM_OK;
}

int64_t tm_selected_page_attention_workspace_size(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                                  int64_t count) {
  report(TM_OK, "%s", "");
  if (check_selected(batch, rows, heads, kv_heads, count) != TM_OK) return -1;
  if (batch == 0 || rows == 0) return 0;
  const RowsPlan plan = selected_plan(batch, rows, heads, kv_heads, count);
  return check_units(plan.units) == TM_OK ? plan.workspace_bytes : -1;
}

int tm_selected_page_attention(const void* query, int64_t query_stride, const void* key_cache,
                               int64_t key_page_stride, const void* value_cache, int64_t value_page_stride,
                               const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens,
                               const int32_t* pages, void* out, int64_t batch, int64_t rows, int64_t heads,
                               int64_t kv_heads, int64_t table_cols, int64_t num_pages, int64_t count, float scale,
                               int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  int st = check_dtype(dtype);
  if (st == TM_OK) st = check_selected(batch, rows, heads, kv_heads, count);
  if (st == TM_OK) st = check_table(table_cols, table_stride, batch);
  if (st == TM_OK) st = check_cache(num_pages, key_page_stride, kv_heads, "key_cache");
  if (st == TM_OK) st = check_cache(num_pages, value_page_stride, kv_heads, "value_cache");
  if (st == TM_OK) st = check_stride(query_stride, heads * tmx::kHeadDim, batch * rows, "query");
  if (st == TM_OK) st = check_scale(scale);
  if (st != TM_OK || batch == 0 || rows == 0) return st;
  st = check_aligned({query, key_cache, value_cache, out});
  if (st == TM_OK) st = check_element(block_table, 4);
  if (st == TM_OK) st = check_element(seq_lens, 4);
  if (st == TM_OK) st = check_element(pages, 4);
  if (st != TM_OK) return st;
  const RowsPlan plan = selected_plan(batch, rows, heads, kv_heads, count);
  st = check_units(plan.units);
  if (st == TM_OK) st = check_workspace(workspace, workspace_bytes, plan.workspace_bytes);
  if (st != TM_OK) return st;
  const int64_t blocks = (rows + tmx::kSelectRows - 1) / tmx::kSelectRows;
  const Range written[] = {{out, batch * rows * heads * kHeadBytes, "out"},
                           {workspace, plan.workspace_bytes, "workspace"}};
  const Range read[] = {{query, rows_bytes(batch * rows, query_stride, heads * tmx::kHeadDim), "query"},
                        {key_cache, cache_bytes(num_pages, key_page_stride, kv_heads), "key_cache"},
                        {value_cache, cache_bytes(num_pages, value_page_stride, kv_heads), "value_cache"},
                        {block_table, table_bytes(batch, table_stride, table_cols), "block_table"},
                        {seq_lens, batch * 4, "seq_lens"},
                        {pages, batch * blocks * kv_heads * count * 4, "pages"}};
  st = check_overlap(written, read);
  if (st != TM_OK) return st;
  tmx::RowsParams p{};
  p.query = static_cast<const uint16_t*>(query);
  p.query_stride = query_stride;
  p.key_cache = static_cast<const char*>(key_cache);
  p.value_cache = static_cast<const char*>(value_cache);
  p.key_page_stride = key_page_stride * 2;
  p.value_page_stride = value_page_stride * 2;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.lens = seq_lens;
  p.selected = pages;
  p.out = static_cast<uint16_t*>(out);
  p.counters = static_cast<unsigned long long*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + tmx::kCounterBytes);
  p.epoch = tmx::workspace_tag(workspace);
  p.table_cols = (int)table_cols;
  p.batch = (int)batch;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads);
  p.num_pages = (int)num_pages;
  p.total_rows = (int)(batch * rows);
  p.rows = (int)rows;
  p.blocks = (int)blocks;
  p.count = (int)count;
  p.workgroups = plan.workgroups;
  p.total_units = (int)plan.units;
  p.per_run = (int)plan.per_run;
  p.scale_log2 = scale * 1.4426950408889634f;
  return launch_attention(p, plan, dtype, stream);
}

int64_t tm_tree_attention_workspace_size(int64_t total_rows, int64_t batch, int64_t heads, int64_t kv_heads,
                                         int64_t table_cols) {
  report(TM_OK, "%s", "");
  if (check_tree(total_rows, batch, heads, kv_heads, table_cols) != TM_OK) return -1;
  if (batch == 0 || total_rows == 0) return 0;
  const RowsPlan plan = tree_plan(total_rows, batch, heads, kv_heads, table_cols);
  return check_units(plan.units) == TM_OK ? plan.workspace_bytes : -1;
}

int tm_tree_attention(const void* query, int64_t query_stride, const void* key, int64_t key_stride,
                      const void* value, int64_t value_stride, const void* key_cache, int64_t key_page_stride,
                      const void* value_cache, int64_t value_page_stride, const int32_t* block_table,
                      int64_t table_stride, const int32_t* context_lens, const int32_t* tree_offsets,
                      const int64_t* tree_mask, void* out, int64_t total_rows, int64_t batch, int64_t heads,
                      int64_t kv_heads, int64_t table_cols, int64_t num_pages, float scale, int dtype,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  int st = check_dtype(dtype);
  if (st == TM_OK) st = check_tree(total_rows, batch, heads, kv_heads, table_cols);
  if (st == TM_OK) st = check_table(table_cols, table_stride, batch);
  if (st == TM_OK) st = check_cache(num_pages, key_page_stride, kv_heads, "key_cache");
  if (st == TM_OK) st = check_cache(num_pages, value_page_stride, kv_heads, "value_cache");
  if (st == TM_OK) st = check_stride(query_stride, heads * tmx::kHeadDim, total_rows, "query");
  if (st == TM_OK) st = check_stride(key_stride, kv_heads * tmx::kHeadDim, total_rows, "key");
  if (st == TM_OK) st = check_stride(value_stride, kv_heads * tmx::kHeadDim, total_rows, "value");
  if (st == TM_OK) st = check_scale(scale);
  if (st != TM_OK || batch == 0 || total_rows == 0) return st;
  st = check_aligned({query, key, value, key_cache, value_cache, out});
  if (st == TM_OK) st = check_element(block_table, 4);
  if (st == TM_OK) st = check_element(context_lens, 4);
  if (st == TM_OK) st = check_element(tree_offsets, 4);
  if (st == TM_OK) st = check_element(tree_mask, 8);
  if (st != TM_OK) return st;
  const RowsPlan plan = tree_plan(total_rows, batch, heads, kv_heads, table_cols);
  st = check_units(plan.units);
  if (st == TM_OK) st = check_workspace(workspace, workspace_bytes, plan.workspace_bytes);
  if (st != TM_OK) return st;
  const Range written[] = {{out, total_rows * heads * kHeadBytes, "out"},
                           {workspace, plan.workspace_bytes, "workspace"}};
  const Range read[] = {{query, rows_bytes(total_rows, query_stride, heads * tmx::kHeadDim), "query"},
                        {key, rows_bytes(total_rows, key_stride, kv_heads * tmx::kHeadDim), "key"},
                        {value, rows_bytes(total_rows, value_stride, kv_heads * tmx::kHeadDim), "value"},
                        {key_cache, cache_bytes(num_pages, key_page_stride, kv_heads), "key_cache"},
                        {value_cache, cache_bytes(num_pages, value_page_stride, kv_heads), "value_cache"},
                        {block_table, table_bytes(batch, table_stride, table_cols), "block_table"},
                        {context_lens, batch * 4, "context_lens"},
                        {tree_offsets, (batch + 1) * 4, "tree_offsets"},
                        {tree_mask, total_rows * 8, "tree_mask"}};
  st = check_overlap(written, read);
  if (st != TM_OK) return st;
  tmx::RowsParams p{};
  p.query = static_cast<const uint16_t*>(query);
  p.query_stride = query_stride;
  p.key_cache = static_cast<const char*>(key_cache);
  p.value_cache = static_cast<const char*>(value_cache);
  p.key_page_stride = key_page_stride * 2;
  p.value_page_stride = value_page_stride * 2;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.lens = context_lens;
  p.draft_key = static_cast<const char*>(key);
  p.draft_value = static_cast<const char*>(value);
  p.draft_key_stride = key_stride * 2;
  p.draft_value_stride = value_stride * 2;
  p.tree_offsets = tree_offsets;
  p.tree_mask = tree_mask;
  p.out = static_cast<uint16_t*>(out);
  p.counters = static_cast<unsigned long long*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + tmx::kCounterBytes);
  p.epoch = tmx::workspace_tag(workspace);
  p.table_cols = (int)table_cols;
  p.batch = (int)batch;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads);
  p.num_pages = (int)num_pages;
  p.total_rows = (int)total_rows;
  p.workgroups = plan.workgroups;
  p.scale_log2 = scale * 1.4426950408889634f;
  return launch_attention(p, plan, dtype, stream);
}

}  // extern "C"
