// Argument checks and accessors that the torch operators of the serving entry
// points share.
#ifndef TRIANGLEMIX_TORCH_CHECKS_H
#define TRIANGLEMIX_TORCH_CHECKS_H

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <initializer_list>

#include "../../include/trianglemix_pages.h"

namespace trianglemix_rocm {

struct Named {
  const at::Tensor& tensor;
  const char* name;
};

inline void check_device(std::initializer_list<Named> all) {
  const at::Tensor& first = all.begin()->tensor;
  for (const Named& n : all) {
    TORCH_CHECK(n.tensor.is_cuda(), n.name, " must be a GPU tensor");
    TORCH_CHECK(n.tensor.device() == first.device(), "all inputs must be on the same GPU device");
  }
}

// TM_BF16 or TM_FP16, shared by all of them.
inline int check_type(std::initializer_list<Named> all) {
  const at::ScalarType type = all.begin()->tensor.scalar_type();
  TORCH_CHECK(type == at::ScalarType::BFloat16 || type == at::ScalarType::Half, all.begin()->name,
              " must be BF16 or FP16");
  for (const Named& n : all) TORCH_CHECK(n.tensor.scalar_type() == type, n.name, " must have the type of ", all.begin()->name);
  return type == at::ScalarType::Half ? TM_FP16 : TM_BF16;
}

// [rows, heads, 128] with contiguous rows.
inline void check_rows(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.dim() == 3 && x.size(2) == 128, name, " must be [rows, heads, 128]");
  TORCH_CHECK(x.numel() == 0 || (x.stride(2) == 1 && (x.size(1) == 1 || x.stride(1) == 128)), "the [heads, 128] part of each ", name,
              " row must be contiguous");
}

// The row stride; that of a single row may be anything.
inline int64_t row_stride(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1) * x.size(2); }

inline void check_cache(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.dim() == 4 && x.size(1) == 128 && x.size(3) == 128, name, " must be [pages, 128, kv_heads, 128]");
  TORCH_CHECK(x.numel() == 0 || (x.stride(3) == 1 && (x.size(2) == 1 || x.stride(2) == 128) && x.stride(1) == 128 * x.size(2)),
              "the pages of ", name, " must be contiguous");
}
inline int64_t page_stride(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : 128 * x.size(2) * 128; }

inline void check_table(const at::Tensor& block_table, const at::Tensor& lens, const char* lens_name) {
  TORCH_CHECK(block_table.scalar_type() == at::ScalarType::Int && block_table.dim() == 2 &&
                  (block_table.numel() == 0 || block_table.size(1) == 1 || block_table.stride(1) == 1),
              "block_table must be an INT32 [batch, max_pages] tensor with contiguous rows");
  TORCH_CHECK(lens.scalar_type() == at::ScalarType::Int && lens.dim() == 1 && lens.is_contiguous(), lens_name,
              " must be a contiguous INT32 [batch] tensor");
  TORCH_CHECK(lens.size(0) == block_table.size(0), lens_name, " must hold one length per row of block_table");
}
inline int64_t table_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Rows per request of a [batch * rows, heads, 128] query.
inline int64_t rows_per_request(const at::Tensor& query, int64_t batch) {
  TORCH_CHECK(batch > 0 ? query.size(0) % batch == 0 : query.size(0) == 0,
              "query must hold the same number of rows for each request");
  return batch > 0 ? query.size(0) / batch : 0;
}

inline void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline void* ptr(const at::Tensor& t) { return t.data_ptr(); }
inline const int32_t* ints(const at::Tensor& t) { return t.data_ptr<int32_t>(); }

}  // namespace trianglemix_rocm

#endif  // TRIANGLEMIX_TORCH_CHECKS_H
