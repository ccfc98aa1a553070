// Torch operators of the paged serving entry points
// (include/trianglemix_pages.h):
//
//   trianglemix::update_page_bounds(key_cache, block_table, seq_lens, num_tokens, page_min!, page_max!) -> ()
//   trianglemix::select_pages(query, page_min, page_max, block_table, seq_lens, count, sink_pages,
//                             recent_pages) -> Tensor, and .out with the count of its out
//   trianglemix::selected_page_attention.out(query, key_cache, value_cache, block_table, seq_lens, pages,
//                                            scale, *, out!), and a functional form
//   trianglemix::tree_attention.out(query, key, value, key_cache, value_cache, block_table, context_lens,
//                                   tree_offsets, tree_mask, scale, *, out!), and a functional form
//
// Shapes, types, devices and overlaps are checked here or in the library, on
// the host; launches go on the current HIP stream of the query's device under
// a device guard, with no synchronisation.  The attention operators, one launch
// each, take the adapter's workspace (trianglemix_torch.cpp); select_pages, which
// keeps scores from one launch to the next, a buffer of each call's own.  The
// functional attention forms return zeros in the rows that the operator leaves
// as they were.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <initializer_list>

#include "../../include/trianglemix_pages.h"
#include "trianglemix_torch.h"

namespace trianglemix_rocm {
namespace {

struct Named {
  const at::Tensor& tensor;
  const char* name;
};

void check_device(std::initializer_list<Named> all) {
  const at::Tensor& first = all.begin()->tensor;
  for (const Named& n : all) {
    TORCH_CHECK(n.tensor.is_cuda(), n.name, " must be a GPU tensor");
    TORCH_CHECK(n.tensor.device() == first.device(), "all inputs must be on the same GPU device");
  }
}

// TM_BF16 or TM_FP16, shared by all of them.
int check_type(std::initializer_list<Named> all) {
  const at::ScalarType type = all.begin()->tensor.scalar_type();
  TORCH_CHECK(type == at::ScalarType::BFloat16 || type == at::ScalarType::Half, all.begin()->name,
              " must be BF16 or FP16");
  for (const Named& n : all) TORCH_CHECK(n.tensor.scalar_type() == type, n.name, " must have the type of ", all.begin()->name);
  return type == at::ScalarType::Half ? TM_FP16 : TM_BF16;
}

// [rows, heads, 128] with contiguous rows.
void check_rows(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.dim() == 3 && x.size(2) == 128, name, " must be [rows, heads, 128]");
  TORCH_CHECK(x.numel() == 0 || (x.stride(2) == 1 && (x.size(1) == 1 || x.stride(1) == 128)), "the [heads, 128] part of each ", name,
              " row must be contiguous");
}

// The row stride; that of a single row may be anything.
int64_t row_stride(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1) * x.size(2); }

void check_cache(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.dim() == 4 && x.size(1) == 128 && x.size(3) == 128, name, " must be [pages, 128, kv_heads, 128]");
  TORCH_CHECK(x.numel() == 0 || (x.stride(3) == 1 && (x.size(2) == 1 || x.stride(2) == 128) && x.stride(1) == 128 * x.size(2)),
              "the pages of ", name, " must be contiguous");
}
int64_t page_stride(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : 128 * x.size(2) * 128; }

void check_table(const at::Tensor& block_table, const at::Tensor& lens, const char* lens_name) {
  TORCH_CHECK(block_table.scalar_type() == at::ScalarType::Int && block_table.dim() == 2 &&
                  (block_table.numel() == 0 || block_table.size(1) == 1 || block_table.stride(1) == 1),
              "block_table must be an INT32 [batch, max_pages] tensor with contiguous rows");
  TORCH_CHECK(lens.scalar_type() == at::ScalarType::Int && lens.dim() == 1 && lens.is_contiguous(), lens_name,
              " must be a contiguous INT32 [batch] tensor");
  TORCH_CHECK(lens.size(0) == block_table.size(0), lens_name, " must hold one length per row of block_table");
}
int64_t table_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void check_bounds(const at::Tensor& page_min, const at::Tensor& page_max, int64_t pages, int64_t kv_heads) {
  TORCH_CHECK(page_min.dim() == 3 && page_min.size(2) == 128 && page_min.is_contiguous(),
              "page_min must be a contiguous [pages, kv_heads, 128] tensor");
  TORCH_CHECK(page_max.sizes() == page_min.sizes() && page_max.is_contiguous(),
              "page_max must be contiguous with the shape of page_min");
  if (pages >= 0) {
    TORCH_CHECK(page_min.size(0) == pages && page_min.size(1) == kv_heads,
                "page_min and page_max must have the pages and KV heads of key_cache");
  }
}

// Rows per request of a [batch * rows, heads, 128] query.
int64_t rows_per_request(const at::Tensor& query, int64_t batch) {
  TORCH_CHECK(batch > 0 ? query.size(0) % batch == 0 : query.size(0) == 0,
              "query must hold the same number of rows for each request");
  return batch > 0 ? query.size(0) / batch : 0;
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void* ptr(const at::Tensor& t) { return t.data_ptr(); }
const int32_t* ints(const at::Tensor& t) { return t.data_ptr<int32_t>(); }

// Of a call's launches.  The stream's shared buffer serves calls of one launch: the
// launches of two host threads on a stream come in any order, so what a launch
// leaves for the next one of its call must be out of the other's reach
// (kPerCall; the caching allocator hands it out again in stream order).
enum class Buffer { kShared, kPerCall };
struct Workspace {
  at::Tensor held;
  void* at = nullptr;
  int64_t bytes = 0;
  Workspace(const at::Tensor& like, int64_t need, void* stream, const char* what, Buffer buffer = Buffer::kShared) {
    TORCH_CHECK(need >= 0, what, " failed (TM_ERR): ", tm_last_error());
    if (need == 0) return;
    held = buffer == Buffer::kPerCall ? at::empty({need}, like.options().dtype(at::kByte))
                                      : workspace_for(like, need, stream);
    at = held.data_ptr();
    bytes = need;
  }
};

}  // namespace

void update_page_bounds(const at::Tensor& key_cache, const at::Tensor& block_table, const at::Tensor& seq_lens,
                        int64_t num_tokens, at::Tensor& page_min, at::Tensor& page_max) {
  check_device({{key_cache, "key_cache"}, {block_table, "block_table"}, {seq_lens, "seq_lens"}, {page_min, "page_min"}, {page_max, "page_max"}});
  const int dtype = check_type({{key_cache, "key_cache"}, {page_min, "page_min"}, {page_max, "page_max"}});
  check_cache(key_cache, "key_cache");
  check_table(block_table, seq_lens, "seq_lens");
  check_bounds(page_min, page_max, key_cache.size(0), key_cache.size(2));
  c10::OptionalDeviceGuard guard(key_cache.device());
  check_status(tm_update_page_bounds(ptr(key_cache), page_stride(key_cache), ints(block_table),
                                     table_stride(block_table), ints(seq_lens), num_tokens, ptr(page_min),
                                     ptr(page_max), block_table.size(0), block_table.size(1), key_cache.size(0),
                                     key_cache.size(2), dtype, stream_of(key_cache)),
               "update_page_bounds");
}

at::Tensor& select_pages_out(const at::Tensor& query, const at::Tensor& page_min, const at::Tensor& page_max,
                             const at::Tensor& block_table, const at::Tensor& seq_lens, int64_t count,
                             int64_t sink_pages, int64_t recent_pages, at::Tensor& out) {
  check_device({{query, "query"}, {page_min, "page_min"}, {page_max, "page_max"}, {block_table, "block_table"}, {seq_lens, "seq_lens"}, {out, "out"}});
  const int dtype = check_type({{query, "query"}, {page_min, "page_min"}, {page_max, "page_max"}});
  check_rows(query, "query");
  check_bounds(page_min, page_max, -1, 0);
  check_table(block_table, seq_lens, "seq_lens");
  const int64_t batch = block_table.size(0), rows = rows_per_request(query, batch);
  const int64_t heads = query.size(1), kv_heads = page_min.size(1);
  TORCH_CHECK(out.scalar_type() == at::ScalarType::Int && out.is_contiguous() && out.dim() == 4 &&
                  out.size(0) == batch && out.size(1) == (rows + TM_SELECT_ROWS - 1) / TM_SELECT_ROWS &&
                  out.size(2) == kv_heads && out.size(3) == count,
              "out must be a contiguous INT32 [batch, ceil(rows / 32), kv_heads, count] tensor");
  c10::OptionalDeviceGuard guard(query.device());
  void* stream = stream_of(query);
  const Workspace ws(query, tm_select_pages_workspace_size(batch, rows, heads, kv_heads, block_table.size(1)), stream,
                     "select_pages", Buffer::kPerCall);
  check_status(tm_select_pages(ptr(query), row_stride(query), ptr(page_min), ptr(page_max), ints(block_table),
                               table_stride(block_table), ints(seq_lens), out.data_ptr<int32_t>(), batch, rows, heads,
                               kv_heads, block_table.size(1), page_min.size(0), count, sink_pages, recent_pages, dtype,
                               ws.at, ws.bytes, stream),
               "select_pages");
  return out;
}

at::Tensor select_pages(const at::Tensor& query, const at::Tensor& page_min, const at::Tensor& page_max,
                        const at::Tensor& block_table, const at::Tensor& seq_lens, int64_t count, int64_t sink_pages,
                        int64_t recent_pages) {
  check_rows(query, "query");
  TORCH_CHECK(block_table.dim() == 2, "block_table must be an INT32 [batch, max_pages] tensor with contiguous rows");
  TORCH_CHECK(page_min.dim() == 3, "page_min must be a contiguous [pages, kv_heads, 128] tensor");
  TORCH_CHECK(count > 0, "count must be positive");
  const int64_t rows = rows_per_request(query, block_table.size(0));
  at::Tensor out = at::empty({block_table.size(0), (rows + TM_SELECT_ROWS - 1) / TM_SELECT_ROWS, page_min.size(1), count},
                             query.options().dtype(at::kInt));
  return select_pages_out(query, page_min, page_max, block_table, seq_lens, count, sink_pages, recent_pages, out);
}

at::Tensor& selected_page_attention_out(const at::Tensor& query, const at::Tensor& key_cache,
                                        const at::Tensor& value_cache, const at::Tensor& block_table,
                                        const at::Tensor& seq_lens, const at::Tensor& pages, double scale,
                                        at::Tensor& out) {
  check_device({{query, "query"}, {key_cache, "key_cache"}, {value_cache, "value_cache"}, {block_table, "block_table"}, {seq_lens, "seq_lens"},
                {pages, "pages"}, {out, "out"}});
  const int dtype = check_type({{query, "query"}, {key_cache, "key_cache"}, {value_cache, "value_cache"}, {out, "out"}});
  check_rows(query, "query");
  check_cache(key_cache, "key_cache");
  check_cache(value_cache, "value_cache");
  TORCH_CHECK(value_cache.sizes() == key_cache.sizes(), "value_cache shape must equal key_cache shape");
  check_table(block_table, seq_lens, "seq_lens");
  const int64_t batch = block_table.size(0), rows = rows_per_request(query, batch);
  const int64_t heads = query.size(1), kv_heads = key_cache.size(2);
  TORCH_CHECK(pages.scalar_type() == at::ScalarType::Int && pages.is_contiguous() && pages.dim() == 4 &&
                  pages.size(0) == batch && pages.size(1) == (rows + TM_SELECT_ROWS - 1) / TM_SELECT_ROWS &&
                  pages.size(2) == kv_heads,
              "pages must be a contiguous INT32 [batch, ceil(rows / 32), kv_heads, count] tensor");
  TORCH_CHECK(out.sizes() == query.sizes() && out.is_contiguous(), "out must be contiguous with the shape of query");
  c10::OptionalDeviceGuard guard(query.device());
  void* stream = stream_of(query);
  const Workspace ws(query, tm_selected_page_attention_workspace_size(batch, rows, heads, kv_heads, pages.size(3)),
                     stream, "selected_page_attention");
  check_status(tm_selected_page_attention(ptr(query), row_stride(query), ptr(key_cache), page_stride(key_cache),
                                          ptr(value_cache), page_stride(value_cache), ints(block_table),
                                          table_stride(block_table), ints(seq_lens), ints(pages), ptr(out), batch,
                                          rows, heads, kv_heads, block_table.size(1), key_cache.size(0),
                                          pages.size(3), static_cast<float>(scale), dtype, ws.at, ws.bytes, stream),
               "selected_page_attention");
  return out;
}

at::Tensor selected_page_attention(const at::Tensor& query, const at::Tensor& key_cache,
                                   const at::Tensor& value_cache, const at::Tensor& block_table,
                                   const at::Tensor& seq_lens, const at::Tensor& pages, double scale) {
  at::Tensor out = at::zeros(query.sizes(), query.options());
  return selected_page_attention_out(query, key_cache, value_cache, block_table, seq_lens, pages, scale, out);
}

at::Tensor& tree_attention_out(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
                               const at::Tensor& key_cache, const at::Tensor& value_cache,
                               const at::Tensor& block_table, const at::Tensor& context_lens,
                               const at::Tensor& tree_offsets, const at::Tensor& tree_mask, double scale,
                               at::Tensor& out) {
  check_device({{query, "query"}, {key, "key"}, {value, "value"}, {key_cache, "key_cache"}, {value_cache, "value_cache"}, {block_table, "block_table"},
                {context_lens, "context_lens"}, {tree_offsets, "tree_offsets"}, {tree_mask, "tree_mask"}, {out, "out"}});
  const int dtype = check_type({{query, "query"}, {key, "key"}, {value, "value"}, {key_cache, "key_cache"}, {value_cache, "value_cache"}, {out, "out"}});
  check_rows(query, "query");
  check_rows(key, "key");
  check_rows(value, "value");
  check_cache(key_cache, "key_cache");
  check_cache(value_cache, "value_cache");
  TORCH_CHECK(value_cache.sizes() == key_cache.sizes(), "value_cache shape must equal key_cache shape");
  check_table(block_table, context_lens, "context_lens");
  const int64_t batch = block_table.size(0), total = query.size(0);
  const int64_t heads = query.size(1), kv_heads = key_cache.size(2);
  TORCH_CHECK(key.size(0) == total && key.size(1) == kv_heads && value.sizes() == key.sizes(),
              "key and value must be [rows, kv_heads, 128] with the rows of query and the KV heads of key_cache");
  TORCH_CHECK(tree_offsets.scalar_type() == at::ScalarType::Int && tree_offsets.dim() == 1 &&
                  tree_offsets.is_contiguous() && tree_offsets.size(0) == batch + 1,
              "tree_offsets must be a contiguous INT32 [batch + 1] tensor");
  TORCH_CHECK(tree_mask.scalar_type() == at::ScalarType::Long && tree_mask.dim() == 1 && tree_mask.is_contiguous() &&
                  tree_mask.size(0) == total,
              "tree_mask must be a contiguous INT64 [rows] tensor");
  TORCH_CHECK(out.sizes() == query.sizes() && out.is_contiguous(), "out must be contiguous with the shape of query");
  c10::OptionalDeviceGuard guard(query.device());
  void* stream = stream_of(query);
  const Workspace ws(query, tm_tree_attention_workspace_size(total, batch, heads, kv_heads, block_table.size(1)), stream,
                     "tree_attention");
  check_status(tm_tree_attention(ptr(query), row_stride(query), ptr(key), row_stride(key), ptr(value),
                                 row_stride(value), ptr(key_cache), page_stride(key_cache), ptr(value_cache),
                                 page_stride(value_cache), ints(block_table), table_stride(block_table),
                                 ints(context_lens), ints(tree_offsets), tree_mask.data_ptr<int64_t>(), ptr(out),
                                 total, batch, heads, kv_heads, block_table.size(1), key_cache.size(0),
                                 static_cast<float>(scale), dtype, ws.at, ws.bytes, stream),
               "tree_attention");
  return out;
}

at::Tensor tree_attention(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value,
                          const at::Tensor& key_cache, const at::Tensor& value_cache, const at::Tensor& block_table,
                          const at::Tensor& context_lens, const at::Tensor& tree_offsets, const at::Tensor& tree_mask,
                          double scale) {
  at::Tensor out = at::zeros(query.sizes(), query.options());
  return tree_attention_out(query, key, value, key_cache, value_cache, block_table, context_lens, tree_offsets,
                            tree_mask, scale, out);
}

namespace {

// Shape-only implementations.
void meta_update_page_bounds(const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, at::Tensor&,
                             at::Tensor&) {}
at::Tensor meta_select_pages(const at::Tensor& query, const at::Tensor& page_min, const at::Tensor&,
                             const at::Tensor& block_table, const at::Tensor&, int64_t count, int64_t, int64_t) {
  const int64_t rows = rows_per_request(query, block_table.size(0));
  return at::empty({block_table.size(0), (rows + TM_SELECT_ROWS - 1) / TM_SELECT_ROWS, page_min.size(1), count},
                   query.options().dtype(at::kInt));
}
at::Tensor& meta_select_pages_out(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                  const at::Tensor&, int64_t, int64_t, int64_t, at::Tensor& out) {
  return out;
}
at::Tensor meta_selected(const at::Tensor& query, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                         const at::Tensor&, const at::Tensor&, double) {
  return at::empty(query.sizes(), query.options());
}
at::Tensor& meta_selected_out(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                              const at::Tensor&, const at::Tensor&, double, at::Tensor& out) {
  return out;
}
at::Tensor meta_tree(const at::Tensor& query, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                     const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                     double) {
  return at::empty(query.sizes(), query.options());
}
at::Tensor& meta_tree_out(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                          const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                          const at::Tensor&, double, at::Tensor& out) {
  return out;
}

}  // namespace
}  // namespace trianglemix_rocm

TORCH_LIBRARY_FRAGMENT(trianglemix, ops) {
  ops.def(
      "update_page_bounds(Tensor key_cache, Tensor block_table, Tensor seq_lens, int num_tokens, "
      "Tensor(a!) page_min, Tensor(b!) page_max) -> ()");
  ops.def(
      "select_pages(Tensor query, Tensor page_min, Tensor page_max, Tensor block_table, Tensor seq_lens, int count, "
      "int sink_pages, int recent_pages) -> Tensor");
  ops.def(
      "select_pages.out(Tensor query, Tensor page_min, Tensor page_max, Tensor block_table, Tensor seq_lens, "
      "int count, int sink_pages, int recent_pages, *, Tensor(a!) out) -> Tensor(a!)");
  ops.def(
      "selected_page_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, "
      "Tensor seq_lens, Tensor pages, float scale) -> Tensor");
  ops.def(
      "selected_page_attention.out(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, "
      "Tensor seq_lens, Tensor pages, float scale, *, Tensor(a!) out) -> Tensor(a!)");
  ops.def(
      "tree_attention(Tensor query, Tensor key, Tensor value, Tensor key_cache, Tensor value_cache, "
      "Tensor block_table, Tensor context_lens, Tensor tree_offsets, Tensor tree_mask, float scale) -> Tensor");
  ops.def(
      "tree_attention.out(Tensor query, Tensor key, Tensor value, Tensor key_cache, Tensor value_cache, "
      "Tensor block_table, Tensor context_lens, Tensor tree_offsets, Tensor tree_mask, float scale, *, "
      "Tensor(a!) out) -> Tensor(a!)");
}

TORCH_LIBRARY_IMPL(trianglemix, CUDA, ops) {
  ops.impl("update_page_bounds", &trianglemix_rocm::update_page_bounds);
  ops.impl("select_pages", &trianglemix_rocm::select_pages);
  ops.impl("select_pages.out", &trianglemix_rocm::select_pages_out);
  ops.impl("selected_page_attention", &trianglemix_rocm::selected_page_attention);
  ops.impl("selected_page_attention.out", &trianglemix_rocm::selected_page_attention_out);
  ops.impl("tree_attention", &trianglemix_rocm::tree_attention);
  ops.impl("tree_attention.out", &trianglemix_rocm::tree_attention_out);
}

TORCH_LIBRARY_IMPL(trianglemix, Meta, ops) {
  ops.impl("update_page_bounds", &trianglemix_rocm::meta_update_page_bounds);
  ops.impl("select_pages", &trianglemix_rocm::meta_select_pages);
  ops.impl("select_pages.out", &trianglemix_rocm::meta_select_pages_out);
  ops.impl("selected_page_attention", &trianglemix_rocm::meta_selected);
  ops.impl("selected_page_attention.out", &trianglemix_rocm::meta_selected_out);
  ops.impl("tree_attention", &trianglemix_rocm::meta_tree);
  ops.impl("tree_attention.out", &trianglemix_rocm::meta_tree_out);
}
