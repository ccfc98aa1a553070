// Host checks and byte counts that the C ABI files of the serving operators
// share.  Each reports through tmx::report and returns the status.
#ifndef TRIANGLEMIX_CHECKS_H
#define TRIANGLEMIX_CHECKS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>
#include <initializer_list>

#include "../../include/trianglemix_pages.h"
#include "trianglemix_pages.h"

namespace tmx {

constexpr int64_t kMaxRows = int64_t(1) << 21;
constexpr int64_t kMaxHeads = 256;
constexpr int64_t kHeadBytes = kHeadDim * 2;

struct Range {
  const void* at;
  int64_t bytes;
  const char* name;
};

inline bool overlap(const Range& a, const Range& b) {
  const uintptr_t x = (uintptr_t)a.at, y = (uintptr_t)b.at;
  return a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}

// What is written must not overlap anything else of the call.
template <size_t W, size_t N>
int check_overlap(const Range (&written)[W], const Range (&read)[N]) {
  for (size_t i = 0; i < W; ++i) {
    for (size_t j = i + 1; j < W; ++j) {
      if (overlap(written[i], written[j])) {
        return report(TM_ERR_INVALID_ARGUMENT, "%s must not overlap %s", written[i].name, written[j].name);
      }
    }
    for (const Range& r : read) {
      if (overlap(written[i], r)) {
        return report(TM_ERR_INVALID_ARGUMENT, "%s must not overlap %s", written[i].name, r.name);
      }
    }
  }
  return TM_OK;
}

// The first check of every entry point: an earlier call's error text goes.
inline int check_dtype(int dtype) {
  report(TM_OK, "%s", "");
  if (dtype != TM_BF16 && dtype != TM_FP16) return report(TM_ERR_INVALID_ARGUMENT, "dtype must be TM_BF16 or TM_FP16");
  return TM_OK;
}

inline int check_heads(int64_t heads, int64_t kv_heads) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) {
    return report(TM_ERR_INVALID_ARGUMENT, "the query heads must be a positive multiple of the KV heads");
  }
  if (heads > kMaxHeads || heads / kv_heads > kMaxGroup) {
    return report(TM_ERR_UNSUPPORTED, "%lld query heads over %lld KV heads; the limits are %lld heads and %d a KV head",
                  (long long)heads, (long long)kv_heads, (long long)kMaxHeads, kMaxGroup);
  }
  return TM_OK;
}

inline int check_batch(int64_t batch, int64_t rows, int64_t total_rows) {
  if (batch < 0 || rows < 0 || total_rows < 0) return report(TM_ERR_INVALID_ARGUMENT, "sizes must not be negative");
  if (batch > kMaxBatch) {
    return report(TM_ERR_UNSUPPORTED, "%lld requests; the limit is %d", (long long)batch, kMaxBatch);
  }
  if (rows > kMaxRows || total_rows > kMaxRows) {
    return report(TM_ERR_UNSUPPORTED, "more than %lld query rows", (long long)kMaxRows);
  }
  return TM_OK;
}

inline int check_table(int64_t table_cols, int64_t table_stride, int64_t batch) {
  if (table_cols <= 0 || (batch > 1 && table_stride < table_cols)) {
    return report(TM_ERR_INVALID_ARGUMENT, "block_table must be [batch, max_pages] with rows that do not overlap");
  }
  if (table_cols > kMaxTableCols) {
    return report(TM_ERR_UNSUPPORTED, "block_table has %lld columns; the limit is %d", (long long)table_cols,
                  kMaxTableCols);
  }
  return TM_OK;
}

inline int check_cache(int64_t num_pages, int64_t page_stride, int64_t kv_heads, const char* name, int elem_bytes = 2) {
  if (num_pages <= 0) return report(TM_ERR_INVALID_ARGUMENT, "%s must be [pages, 128, kv_heads, 128] with pages > 0", name);
  if (num_pages > kMaxPages) {
    return report(TM_ERR_UNSUPPORTED, "%s has %lld pages; the limit is %lld", name, (long long)num_pages,
                  (long long)kMaxPages);
  }
  const int64_t page = kPageSize * kv_heads * kHeadDim;
  if (page_stride < page || page_stride * elem_bytes % 16 != 0 || page_stride > (int64_t(1) << 40)) {
    return report(TM_ERR_INVALID_ARGUMENT,
                  "%s pages must be contiguous with a page stride of at least a page that is a multiple of %d", name,
                  16 / elem_bytes);
  }
  return TM_OK;
}

inline int check_stride(int64_t stride, int64_t width, int64_t rows, const char* name) {
  if ((rows > 1 && stride < width) || stride < 0 || stride % 8 != 0 || stride > (int64_t(1) << 23)) {
    return report(TM_ERR_INVALID_ARGUMENT,
                  "%s rows must hold [heads, 128] contiguous elements with a row stride that is a multiple of 8", name);
  }
  return TM_OK;
}

inline int check_aligned(std::initializer_list<const void*> pointers) {
  for (const void* p : pointers) {
    if (!p) return report(TM_ERR_INVALID_ARGUMENT, "tensors must be non-null");
    if ((uintptr_t)p & 15) return report(TM_ERR_INVALID_ARGUMENT, "tensors must be 16-byte aligned");
  }
  return TM_OK;
}

// Tables, lengths, masks and lists are read (written) element by element.
inline int check_element(const void* p, uintptr_t bytes) {
  if (!p) return report(TM_ERR_INVALID_ARGUMENT, "tensors must be non-null");
  if ((uintptr_t)p & (bytes - 1)) return report(TM_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
  return TM_OK;
}

inline int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
  if (bytes < 0 || (bytes > 0 && !workspace)) return report(TM_ERR_WORKSPACE, "workspace pointer/size are inconsistent");
  if (bytes < need) {
    return report(TM_ERR_WORKSPACE, "workspace of %lld bytes is smaller than the %lld bytes this call needs",
                  (long long)bytes, (long long)need);
  }
  if ((uintptr_t)workspace & 15) return report(TM_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  return TM_OK;
}

inline int check_scale(float scale) {
  if (!std::isfinite(scale) || scale <= 0.0f) return report(TM_ERR_INVALID_ARGUMENT, "scale must be finite and positive");
  return TM_OK;
}

inline int launched(hipError_t err) {
  if (err == hipSuccess) return TM_OK;
  return report(TM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
}

inline int64_t cache_bytes(int64_t num_pages, int64_t page_stride, int64_t kv_heads, int elem_bytes = 2) {
  return ((num_pages - 1) * page_stride + kPageSize * kv_heads * kHeadDim) * elem_bytes;
}
inline int64_t rows_bytes(int64_t rows, int64_t stride, int64_t width) { return rows > 0 ? ((rows - 1) * stride + width) * 2 : 0; }
inline int64_t table_bytes(int64_t batch, int64_t stride, int64_t cols) { return batch > 0 ? ((batch - 1) * stride + cols) * 4 : 0; }

inline int check_units(int64_t units) {
  if (units > kMaxUnits) {
    return report(TM_ERR_UNSUPPORTED, "the call may read %lld pages of 128 keys; the limit is %d", (long long)units,
                  kMaxUnits);
  }
  return TM_OK;
}

}  // namespace tmx

#endif  // TRIANGLEMIX_CHECKS_H
