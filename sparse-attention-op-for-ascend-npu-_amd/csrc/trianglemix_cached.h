// Internal interface of the cached-attention operators (position rotation,
// rotated cache write, attention over the cache) between their host code and
// their kernels.
#ifndef TRIANGLEMIX_CACHED_INTERNAL_H
#define TRIANGLEMIX_CACHED_INTERNAL_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "trianglemix_kernel.h"
#include "trianglemix_pages.h"

namespace tmx {

enum class CacheType { kSame, kE4m3 };  // of the rows' own type, or 8-bit with a scale for each KV head

struct RotateParams {
  const uint16_t* query;  // [rows, heads, 128]
  const uint16_t* key;    // [rows, kv_heads, 128]
  const uint16_t* value;
  uint16_t* query_out;
  int64_t query_stride, key_stride, value_stride, out_stride;  // elements
  const int64_t* positions;
  const int64_t* slots;
  const double* frequencies;
  char* key_cache;
  char* value_cache;
  int64_t key_page_stride, value_page_stride;  // bytes
  const float* key_scale;
  const float* value_scale;
  int64_t num_slots;
  int rows, heads, kv_heads;  // kv_heads 0: rotation alone
  int rotary_dim;
  float magnitude;
};
hipError_t launch_rotate(const RotateParams& p, bool interleaved, bool fp16, CacheType cache, hipStream_t stream);

struct CachedParams {
  const uint16_t* query;  // [batch * rows, heads, 128]
  int64_t query_stride;   // elements
  const char* key_cache;
  const char* value_cache;
  int64_t key_page_stride, value_page_stride;  // bytes
  const float* key_scale;                      // [kv_heads], or null
  const float* value_scale;
  const int32_t* block_table;
  int64_t table_stride;
  const int32_t* seq_lens;
  uint16_t* out;  // [batch * rows, heads, 128]
  unsigned long long* counters;
  float* partials;
  unsigned long long epoch;
  int table_cols, batch, rows, heads, kv_heads, group, num_pages;
  int window, sinks;  // window -1: all keys
  // Few rows: the waves of a workgroup, 2^row_shift row tiles times 2^key_shift parts of
  // the keys times as many KV heads as that leaves.
  int row_shift, key_shift;
  int full_shares, min_tiles;  // shares of the keys, of at least min_tiles tiles, by the requests' lengths,
  int halvings;                // made even by so many steps
  // Chunks: tokens of a workgroup's rows, how many such parts a request has; of all
  // requests' parts, the latest first, full_parts have a workgroup a KV head, the
  // others one for each of `splits` shares of their keys.
  int part_tokens, row_parts, full_parts, splits;
  int workgroups;              // of the grid
  float scale_log2;
};
// A wave's rows and a workgroup's waves: 16 x 4, 16 x 8 or 32 x 8.
struct CachedShape {
  int rows, waves;
};
// Chunks, of more rows of a KV head than most_few_rows: workgroups of kChunkRows rows or
// of half as many.  (32 requests of 32 tokens, four heads a KV head, 500 to 9000 tokens
// before them: 128 rows a workgroup that loads for itself 233 us, as chunks 178.  Of 16
// tokens, 64 rows, 115 and 173 over 8-bit caches, 185 and 178 over 16-bit ones, whose tiles
// fill the registers; 64 of up to 3000 tokens 110 | 124 and 167 | 131.)
constexpr int kChunkRows = 256;
// Steps of 64 keys that a share of a part has at least, also where the requests are far
// shorter than their table is wide (16384 columns, one request: 128 rows of 300 tokens 24
// us, without a least 30, with eight steps 20; but 75 rows of 3000 tokens 36, with eight
// 42.  In tables as wide as the request is long they take 17 and 27).
constexpr int kLeastSteps = 4;
constexpr int most_few_rows(CacheType type) { return type == CacheType::kE4m3 ? 64 : 32; }
hipError_t launch_cached_chunks(const CachedParams& p, int rows, bool fp16, CacheType cache, hipStream_t stream);
hipError_t launch_cached_attention(const CachedParams& p, CachedShape shape, bool fp16, CacheType cache,
                                   hipStream_t stream);

}  // namespace tmx

#endif  // TRIANGLEMIX_CACHED_INTERNAL_H
