// Torch operators of the cached-attention entry points
// (include/trianglemix_cached.h):
//
//   trianglemix::rotate_positions(x, positions, frequencies, interleaved, magnitude) -> Tensor, and .out
//   trianglemix::rotate_and_cache(query, key, value, positions, slot_mapping, frequencies, interleaved, magnitude,
//                                 query_out!, key_cache!, value_cache!, key_scale, value_scale) -> ()
//   trianglemix::cached_attention(query, key_cache, value_cache, block_table, seq_lens, scale, window, sinks,
//                                 key_scale, value_scale) -> Tensor, and .out
//
// Shapes, types, devices and overlaps are checked here or in the library, on
// the host; launches go on the current HIP stream of the first tensor's device
// under a device guard, with no synchronisation.  cached_attention, one launch,
// takes the adapter's workspace (trianglemix_torch.cpp).  The functional forms
// return zeros in the rows that the operator leaves as they were.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <optional>

#include "../../include/trianglemix_cached.h"
#include "trianglemix_torch.h"
#include "trianglemix_torch_checks.h"

namespace trianglemix_rocm {
namespace {

typedef std::optional<at::Tensor> MaybeTensor;

void check_positions(const at::Tensor& positions, const at::Tensor& frequencies, const at::Tensor& x) {
  TORCH_CHECK(positions.scalar_type() == at::ScalarType::Long && positions.dim() == 1 && positions.is_contiguous() &&
                  positions.size(0) == x.size(0),
              "positions must be a contiguous INT64 [rows] tensor");
  TORCH_CHECK(frequencies.scalar_type() == at::ScalarType::Double && frequencies.dim() == 1 && frequencies.is_contiguous(),
              "frequencies must be a contiguous FP64 [rotary_dim / 2] tensor");
}

// The caches' type (TM_BF16, TM_FP16 or TM_E4M3) with what belongs to it.
int check_caches(const at::Tensor& rows, const at::Tensor& key_cache, const at::Tensor& value_cache,
                 const MaybeTensor& key_scale, const MaybeTensor& value_scale) {
  check_cache(key_cache, "key_cache");
  check_cache(value_cache, "value_cache");
  TORCH_CHECK(value_cache.sizes() == key_cache.sizes(), "value_cache shape must equal key_cache shape");
  TORCH_CHECK(value_cache.scalar_type() == key_cache.scalar_type(), "value_cache must have the type of key_cache");
  const bool e4m3 = key_cache.scalar_type() == at::ScalarType::Float8_e4m3fn;
  TORCH_CHECK(e4m3 || key_cache.scalar_type() == rows.scalar_type(), "the caches must be FP8 (e4m3fn) or have the type of query");
  TORCH_CHECK(key_scale.has_value() == e4m3 && value_scale.has_value() == e4m3,
              "key_scale and value_scale belong to FP8 caches, and only to them");
  if (!e4m3) return rows.scalar_type() == at::ScalarType::Half ? TM_FP16 : TM_BF16;
  for (const at::Tensor& s : {*key_scale, *value_scale}) {
    TORCH_CHECK(s.scalar_type() == at::ScalarType::Float && s.dim() == 1 && s.is_contiguous() && s.size(0) == key_cache.size(2),
                "key_scale and value_scale must be contiguous FP32 [kv_heads] tensors");
    check_device({{rows, "query"}, {s, "key_scale and value_scale"}});
  }
  return TM_E4M3;
}

const float* scales(const MaybeTensor& s) { return s.has_value() ? s->data_ptr<float>() : nullptr; }

}  // namespace

at::Tensor& rotate_positions_out(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& frequencies,
                                 bool interleaved, double magnitude, at::Tensor& out) {
  check_device({{x, "x"}, {positions, "positions"}, {frequencies, "frequencies"}, {out, "out"}});
  const int dtype = check_type({{x, "x"}, {out, "out"}});
  check_rows(x, "x");
  check_rows(out, "out");
  TORCH_CHECK(out.sizes() == x.sizes(), "out must have the shape of x");
  check_positions(positions, frequencies, x);
  c10::OptionalDeviceGuard guard(x.device());
  check_status(tm_rotate_positions(ptr(x), row_stride(x), positions.data_ptr<int64_t>(), frequencies.data_ptr<double>(),
                                   ptr(out), row_stride(out), x.size(0), x.size(1), 2 * frequencies.size(0), interleaved,
                                   static_cast<float>(magnitude), dtype, stream_of(x)),
               "rotate_positions");
  return out;
}

at::Tensor rotate_positions(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& frequencies,
                            bool interleaved, double magnitude) {
  at::Tensor out = at::zeros(x.sizes(), x.options());
  return rotate_positions_out(x, positions, frequencies, interleaved, magnitude, out);
}

void rotate_and_cache(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value, const at::Tensor& positions,
                      const at::Tensor& slot_mapping, const at::Tensor& frequencies, bool interleaved, double magnitude,
                      at::Tensor& query_out, at::Tensor& key_cache, at::Tensor& value_cache, const MaybeTensor& key_scale,
                      const MaybeTensor& value_scale) {
  check_device({{query, "query"}, {key, "key"}, {value, "value"}, {positions, "positions"}, {slot_mapping, "slot_mapping"},
                {frequencies, "frequencies"}, {query_out, "query_out"}, {key_cache, "key_cache"}, {value_cache, "value_cache"}});
  const int dtype = check_type({{query, "query"}, {key, "key"}, {value, "value"}, {query_out, "query_out"}});
  check_rows(query, "query");
  check_rows(key, "key");
  check_rows(value, "value");
  check_rows(query_out, "query_out");
  TORCH_CHECK(query_out.sizes() == query.sizes(), "query_out must have the shape of query");
  const int cache_dtype = check_caches(query, key_cache, value_cache, key_scale, value_scale);
  const int64_t rows = query.size(0), heads = query.size(1), kv_heads = key_cache.size(2);
  TORCH_CHECK(key.size(0) == rows && key.size(1) == kv_heads && value.sizes() == key.sizes(),
              "key and value must be [rows, kv_heads, 128] with the rows of query and the KV heads of key_cache");
  check_positions(positions, frequencies, query);
  TORCH_CHECK(slot_mapping.scalar_type() == at::ScalarType::Long && slot_mapping.dim() == 1 &&
                  slot_mapping.is_contiguous() && slot_mapping.size(0) == rows,
              "slot_mapping must be a contiguous INT64 [rows] tensor");
  c10::OptionalDeviceGuard guard(query.device());
  check_status(tm_rotate_and_cache(ptr(query), row_stride(query), ptr(key), row_stride(key), ptr(value), row_stride(value),
                                   positions.data_ptr<int64_t>(), slot_mapping.data_ptr<int64_t>(),
                                   frequencies.data_ptr<double>(), ptr(query_out), row_stride(query_out), ptr(key_cache),
                                   page_stride(key_cache), ptr(value_cache), page_stride(value_cache), scales(key_scale),
                                   scales(value_scale), rows, heads, kv_heads, key_cache.size(0), 2 * frequencies.size(0),
                                   interleaved, static_cast<float>(magnitude), dtype, cache_dtype, stream_of(query)),
               "rotate_and_cache");
}

at::Tensor& cached_attention_out(const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
                                 const at::Tensor& block_table, const at::Tensor& seq_lens, double scale, int64_t window,
                                 int64_t sinks, const MaybeTensor& key_scale, const MaybeTensor& value_scale,
                                 at::Tensor& out) {
  check_device({{query, "query"}, {key_cache, "key_cache"}, {value_cache, "value_cache"}, {block_table, "block_table"},
                {seq_lens, "seq_lens"}, {out, "out"}});
  const int dtype = check_type({{query, "query"}, {out, "out"}});
  check_rows(query, "query");
  const int cache_dtype = check_caches(query, key_cache, value_cache, key_scale, value_scale);
  check_table(block_table, seq_lens, "seq_lens");
  const int64_t batch = block_table.size(0), rows = rows_per_request(query, batch);
  const int64_t heads = query.size(1), kv_heads = key_cache.size(2);
  TORCH_CHECK(out.sizes() == query.sizes() && out.is_contiguous(), "out must be contiguous with the shape of query");
  c10::OptionalDeviceGuard guard(query.device());
  void* stream = stream_of(query);
  const int64_t need = tm_cached_attention_workspace_size(batch, rows, heads, kv_heads, block_table.size(1), window, sinks);
  TORCH_CHECK(need >= 0, "cached_attention failed (TM_ERR): ", tm_last_error());
  at::Tensor workspace;
  if (need > 0) workspace = workspace_for(query, need, stream);
  check_status(tm_cached_attention(ptr(query), row_stride(query), ptr(key_cache), page_stride(key_cache), ptr(value_cache),
                                   page_stride(value_cache), scales(key_scale), scales(value_scale), ints(block_table),
                                   table_stride(block_table), ints(seq_lens), ptr(out), batch, rows, heads, kv_heads,
                                   block_table.size(1), key_cache.size(0), window, sinks, static_cast<float>(scale), dtype,
                                   cache_dtype, need > 0 ? ptr(workspace) : nullptr, need, stream),
               "cached_attention");
  return out;
}

at::Tensor cached_attention(const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
                            const at::Tensor& block_table, const at::Tensor& seq_lens, double scale, int64_t window,
                            int64_t sinks, const MaybeTensor& key_scale, const MaybeTensor& value_scale) {
  at::Tensor out = at::zeros(query.sizes(), query.options());
  return cached_attention_out(query, key_cache, value_cache, block_table, seq_lens, scale, window, sinks, key_scale,
                              value_scale, out);
}

namespace {

// Shape-only implementations.
at::Tensor meta_rotate(const at::Tensor& x, const at::Tensor&, const at::Tensor&, bool, double) {
  return at::empty(x.sizes(), x.options());
}
at::Tensor& meta_rotate_out(const at::Tensor&, const at::Tensor&, const at::Tensor&, bool, double, at::Tensor& out) {
  return out;
}
void meta_rotate_and_cache(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                           const at::Tensor&, bool, double, at::Tensor&, at::Tensor&, at::Tensor&, const MaybeTensor&,
                           const MaybeTensor&) {}
at::Tensor meta_cached(const at::Tensor& query, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                       double, int64_t, int64_t, const MaybeTensor&, const MaybeTensor&) {
  return at::empty(query.sizes(), query.options());
}
at::Tensor& meta_cached_out(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            double, int64_t, int64_t, const MaybeTensor&, const MaybeTensor&, at::Tensor& out) {
  return out;
}

}  // namespace
}  // namespace trianglemix_rocm

TORCH_LIBRARY_FRAGMENT(trianglemix, ops) {
  ops.def(
      "rotate_positions(Tensor x, Tensor positions, Tensor frequencies, bool interleaved, float magnitude) -> Tensor");
  ops.def(
      "rotate_positions.out(Tensor x, Tensor positions, Tensor frequencies, bool interleaved, float magnitude, *, "
      "Tensor(a!) out) -> Tensor(a!)");
  ops.def(
      "rotate_and_cache(Tensor query, Tensor key, Tensor value, Tensor positions, Tensor slot_mapping, "
      "Tensor frequencies, bool interleaved, float magnitude, Tensor(a!) query_out, Tensor(b!) key_cache, "
      "Tensor(c!) value_cache, Tensor? key_scale=None, Tensor? value_scale=None) -> ()");
  ops.def(
      "cached_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, "
      "float scale, int window=-1, int sinks=0, Tensor? key_scale=None, Tensor? value_scale=None) -> Tensor");
  ops.def(
      "cached_attention.out(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, "
      "float scale, int window=-1, int sinks=0, Tensor? key_scale=None, Tensor? value_scale=None, *, "
      "Tensor(a!) out) -> Tensor(a!)");
}

TORCH_LIBRARY_IMPL(trianglemix, CUDA, ops) {
  ops.impl("rotate_positions", &trianglemix_rocm::rotate_positions);
  ops.impl("rotate_positions.out", &trianglemix_rocm::rotate_positions_out);
  ops.impl("rotate_and_cache", &trianglemix_rocm::rotate_and_cache);
  ops.impl("cached_attention", &trianglemix_rocm::cached_attention);
  ops.impl("cached_attention.out", &trianglemix_rocm::cached_attention_out);
}

TORCH_LIBRARY_IMPL(trianglemix, Meta, ops) {
  ops.impl("rotate_positions", &trianglemix_rocm::meta_rotate);
  ops.impl("rotate_positions.out", &trianglemix_rocm::meta_rotate_out);
  ops.impl("rotate_and_cache", &trianglemix_rocm::meta_rotate_and_cache);
  ops.impl("cached_attention", &trianglemix_rocm::meta_cached);
  ops.impl("cached_attention.out", &trianglemix_rocm::meta_cached_out);
}
