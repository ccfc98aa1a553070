// C ABI of the cached-attention operators (include/trianglemix_cached.h): host
// checks and launch geometry.  Every check runs before any HIP call.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <array>

#include "../../include/trianglemix_cached.h"
#include "trianglemix_cached.h"
#include "trianglemix_checks.h"

namespace {

using namespace tmx;

// Rows of `width` bytes, `stride` bytes apart.
struct Rows {
  const void* at;
  int64_t stride, width, rows;
  const char* name;
  Range range() const { return {at, rows > 0 ? (rows - 1) * stride + width : 0, name}; }
};

// Views of one buffer whose rows lie side by side (a fused projection) do not
// overlap, though their ranges do.
bool overlap(const Rows& a, const Rows& b) {
  if (!tmx::overlap(a.range(), b.range())) return false;
  if (a.rows == 1 && b.rows == 1) return true;
  const int64_t stride = a.rows > 1 ? a.stride : b.stride;
  if (stride <= 0 || (a.rows > 1 && b.rows > 1 && a.stride != b.stride)) return true;
  const int64_t apart = (int64_t)((uintptr_t)b.at - (uintptr_t)a.at) % stride;
  const int64_t behind = apart < 0 ? apart + stride : apart;  // b's rows begin so far behind a's
  return behind < a.width || behind + b.width > stride;
}

bool same(const Rows& a, const Rows& b) { return a.at == b.at && (a.rows <= 1 || a.stride == b.stride); }

int refuse_overlap(const char* a, const char* b) {
  return report(TM_ERR_INVALID_ARGUMENT, "%s must not overlap %s", a, b);
}

int check_rotation(int64_t rows, int64_t rotary_dim, float magnitude) {
  if (rows < 0) return report(TM_ERR_INVALID_ARGUMENT, "sizes must not be negative");
  if (rows > kMaxRows) return report(TM_ERR_UNSUPPORTED, "more than %lld rows", (long long)kMaxRows);
  if (rotary_dim < 16 || rotary_dim > kHeadDim || rotary_dim % 16 != 0) {
    return report(TM_ERR_UNSUPPORTED, "rotary_dim must be a multiple of 16 from 16 to %d", kHeadDim);
  }
  if (!std::isfinite(magnitude)) return report(TM_ERR_INVALID_ARGUMENT, "magnitude must be finite");
  return TM_OK;
}

// The cache's type and scales.
int check_cache_type(int dtype, int cache_dtype, const void* key_scale, const void* value_scale, CacheType* type) {
  *type = cache_dtype == TM_E4M3 ? CacheType::kE4m3 : CacheType::kSame;
  if (cache_dtype != TM_E4M3 && cache_dtype != dtype) {
    return report(TM_ERR_INVALID_ARGUMENT, "the caches must hold numbers of the rows' type or TM_E4M3 ones");
  }
  if (cache_dtype == TM_E4M3) {
    int st = check_element(key_scale, 4);
    return st == TM_OK ? check_element(value_scale, 4) : st;
  }
  if (key_scale || value_scale) return report(TM_ERR_INVALID_ARGUMENT, "caches of the rows' type have no scales");
  return TM_OK;
}

int elem_bytes(CacheType type) { return type == CacheType::kE4m3 ? 1 : 2; }

// Partial records of the groups that are cut.
constexpr int64_t kMaxRecordBytes = int64_t(64) << 20;

struct CachedPlan {
  CachedShape shape;
  int row_shift, key_shift, part_tokens, row_parts, full_parts, splits, full_shares, min_tiles, halvings, workgroups;
  int64_t tiles, workspace_bytes;
};

int check_cached(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_cols, int64_t window,
                 int64_t sinks) {
  int st = check_batch(batch, rows, batch * std::max<int64_t>(rows, 0));
  if (st == TM_OK) st = check_heads(heads, kv_heads);
  if (st == TM_OK) st = check_table(table_cols, table_cols, batch);
  if (st != TM_OK) return st;
  if (window < -1 || sinks < 0 || (window == -1 && sinks != 0)) {
    return report(TM_ERR_INVALID_ARGUMENT, "window must be -1 (all keys, sinks 0) or more, sinks must not be negative");
  }
  return TM_OK;
}

// The 32-key tiles that a request's rows can attend at most.
int64_t most_tiles(int64_t rows, int64_t table_cols, int64_t window, int64_t sinks) {
  const int64_t all = table_cols * (kPageSize / kKvTile);
  if (window < 0 || window >= table_cols * kPageSize) return all;
  return std::min(all, (window + rows - 1) / kKvTile + 2 + (std::min(sinks, table_cols * kPageSize) + kKvTile - 1) / kKvTile);
}

CachedPlan cached_plan(CacheType type, int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t table_cols,
                       int64_t window, int64_t sinks) {
  CachedPlan r{};
  const int64_t group = heads / kv_heads, group_rows = rows * group;
  const int64_t tiles = most_tiles(rows, table_cols, window, sinks);
  // Whether groups of 2^shift heads leave every CU 32 tiles.
  const auto enough = [&](int shift) {
    return kv_heads % (1 << shift) == 0 && batch * (kv_heads >> shift) * std::max<int64_t>(1, tiles / 32) >= kComputeUnits;
  };
  if (group_rows > most_few_rows(type)) {
    // Chunks: workgroups of 256 rows, or of 128 with two key parts, one a CU.  What does
    // not fill the GPU's last round is shared out.  Taken is what ends soonest by the
    // time of a step of 64 keys and what a share costs besides (its partial and the merge),
    // in 0.1 us; what every call costs (launch, start, results) is left out on both sides.
    // Lengths are not known here: a request counts as long as its table is wide.
    // 256 | 128 rows, four heads to each of eight KV heads: 33
    // tokens of 8192 40 | 32 us, 75 of 3000 36 | 28, 512 of 8192 88 | 100, 1000 of 20000
    // 326 | 389, 2048 of 32749 1032 | 1220.
    int64_t best = INT64_MAX;
    for (const auto [most_rows, step, besides] : {std::array{kChunkRows, 20, 120}, std::array{kChunkRows / 2, 14, 60}}) {
      const int64_t part_tokens = most_rows / group, row_parts = (rows + part_tokens - 1) / part_tokens;
      const int64_t tiles = most_tiles(part_tokens, table_cols, window, sinks), steps = (tiles + 1) / 2;
      const int64_t parts = batch * row_parts;
      const int64_t rounds = parts * kv_heads / kComputeUnits;  // full ones, to a part: the last may leave CUs to the rest
      const int64_t full_parts = rounds * kComputeUnits / kv_heads;
      const int64_t rest = (parts - full_parts) * kv_heads;
      const int64_t record_bytes = part_tokens * group * (kHeadDim + 2) * 4;
      const int64_t most = std::clamp<int64_t>(rest > 0 ? kMaxRecordBytes / (rest * record_bytes) : 1, 1,
                                               std::clamp<int64_t>(steps / kLeastSteps, 1, 32));
      for (int64_t s = 1; s <= most; ++s) {
        const int64_t rest_rounds = (rest * s + kComputeUnits - 1) / kComputeUnits;
        const int64_t time = rounds * steps * step + rest_rounds * ((steps + s - 1) / s * step + (s > 1 ? besides : 0));
        if (time >= best) continue;
        best = time;
        r.shape.rows = most_rows;
        r.part_tokens = (int)part_tokens;
        r.row_parts = (int)row_parts;
        r.full_parts = (int)full_parts;
        r.splits = (int)s;
        r.tiles = parts * kv_heads * tiles;
        r.workgroups = (int)(full_parts * kv_heads + rest * s);
        r.workspace_bytes = s > 1 ? kCounterBytes + rest * s * record_bytes : 0;
      }
    }
    return r;
  }
  // A wave's rows and the row tiles of a workgroup's waves; what these leave of the
  // waves goes to neighbouring KV heads, whose numbers lie side by side in memory (64
  // requests of 2000 to 16384 tokens: 219 us with eight heads a workgroup, 232 with
  // four, 275 with two), or to parts of the keys: where there is little to read or
  // many rows, whose partials would cost more (32 requests of 5 tokens, 500 to 9000
  // before them: 91 us with eight heads, 75 with four, 79 with two).  So it is with five
  // to sixteen rows of a head: four waves | eight, 32 requests of 4 tokens and of 500 to
  // 9000 69 | 78 us, 1000 of a token and 100 to 900 with eight query heads a KV head 223 |
  // 233; only of many long ones eight take less (64 of 4 tokens, 2000 to 16384: 242 | 231).
  int most_shift;
  if (group_rows <= 16) {
    r.shape = {16, group_rows <= 4 && enough(3) && batch * kv_heads >= kComputeUnits ? 8 : 4};
    most_shift = r.shape.waves == 8 ? 3 : 2;
  } else {
    r.shape = {32, 8};
    r.row_shift = group_rows <= 32 ? 0 : 1;
    most_shift = 2 - r.row_shift;
  }
  int head_shift = 0;
  while (head_shift < most_shift && enough(head_shift + 1)) ++head_shift;
  r.key_shift = (r.shape.waves == 8 ? 3 : 2) - r.row_shift - head_shift;
  const int64_t groups = batch * (kv_heads >> head_shift);
  r.tiles = groups * tiles;
  const int64_t slot_rows = r.row_shift > 0 ? r.shape.rows : std::min<int64_t>(r.shape.rows, group_rows);
  const int64_t record_bytes = (slot_rows << (r.row_shift + head_shift)) * (kHeadDim + 2) * 4;
  const auto grid = [](int64_t shares) { return (shares + 7) / 8 * 8; };  // each workgroup has a record and a word
  int64_t shares = groups;
  r.full_shares = (int)std::max(kComputeUnits - groups, int64_t(kComputeUnits / 2));
  const int64_t most = grid(groups + r.full_shares);
  if (most * record_bytes <= kMaxRecordBytes && most <= kCounterBytes / 8) {
    r.min_tiles = 1 << r.key_shift;
    // Half a microsecond, where the groups are so many that their last shares matter (32
    // requests of 5 tokens 77 us without, 75 with; of 16 tokens 143 and 115).
    r.halvings = tiles > 64 && groups >= kComputeUnits / 4 ? 5 : 0;
    shares = std::min(groups + r.full_shares, r.tiles);
  } else {
    r.min_tiles = (int)tiles;  // no group is cut
  }
  r.workgroups = (int)grid(shares);
  r.workspace_bytes = shares > groups ? kCounterBytes + r.workgroups * record_bytes : 0;
  return r;
}

int check_tiles(int64_t tiles) {
  if (tiles > kMaxUnits) {
    return report(TM_ERR_UNSUPPORTED, "the call may read %lld tiles of 32 keys; the limit is %d", (long long)tiles, kMaxUnits);
  }
  return TM_OK;
}

}  // namespace

extern "C" {

int tm_rotate_positions(const void* x, int64_t x_stride, const int64_t* positions, const double* frequencies,
                        void* out, int64_t out_stride, int64_t rows, int64_t heads, int64_t rotary_dim,
                        int interleaved, float magnitude, int dtype, void* stream) {
  int st = check_dtype(dtype);
  if (st == TM_OK) st = check_rotation(rows, rotary_dim, magnitude);
  if (st == TM_OK) st = check_heads(heads, heads);
  if (st == TM_OK) st = check_stride(x_stride, heads * kHeadDim, rows, "x");
  if (st == TM_OK) st = check_stride(out_stride, heads * kHeadDim, rows, "out");
  if (st != TM_OK || rows == 0) return st;
  st = check_aligned({x, out});
  if (st == TM_OK) st = check_element(positions, 8);
  if (st == TM_OK) st = check_element(frequencies, 8);
  if (st != TM_OK) return st;
  const Rows from{x, x_stride * 2, heads * kHeadBytes, rows, "x"}, to{out, out_stride * 2, heads * kHeadBytes, rows, "out"};
  if (!same(from, to) && overlap(to, from)) return refuse_overlap("out", "x");
  const Range written[] = {to.range()};
  const Range read[] = {{positions, rows * 8, "positions"}, {frequencies, rotary_dim / 2 * 8, "frequencies"}};
  st = check_overlap(written, read);
  if (st != TM_OK) return st;
  RotateParams p{};
  p.query = static_cast<const uint16_t*>(x);
  p.query_out = static_cast<uint16_t*>(out);
  p.query_stride = x_stride;
  p.out_stride = out_stride;
  p.positions = positions;
  p.frequencies = frequencies;
  p.rows = (int)rows;
  p.heads = (int)heads;
  p.rotary_dim = (int)rotary_dim;
  p.magnitude = magnitude;
  return launched(launch_rotate(p, interleaved != 0, dtype == TM_FP16, CacheType::kSame, static_cast<hipStream_t>(stream)));
}

int tm_rotate_and_cache(const void* query, int64_t query_stride, const void* key, int64_t key_stride,
                        const void* value, int64_t value_stride, const int64_t* positions,
                        const int64_t* slot_mapping, const double* frequencies, void* query_out,
                        int64_t query_out_stride, void* key_cache, int64_t key_page_stride, void* value_cache,
                        int64_t value_page_stride, const float* key_scale, const float* value_scale, int64_t rows,
                        int64_t heads, int64_t kv_heads, int64_t num_pages, int64_t rotary_dim, int interleaved,
                        float magnitude, int dtype, int cache_dtype, void* stream) {
  int st = check_dtype(dtype);
  if (st == TM_OK) st = check_rotation(rows, rotary_dim, magnitude);
  if (st == TM_OK) st = check_heads(heads, kv_heads);
  CacheType type;
  if (st == TM_OK) st = check_cache_type(dtype, cache_dtype, key_scale, value_scale, &type);
  if (st == TM_OK) st = check_cache(num_pages, key_page_stride, kv_heads, "key_cache", elem_bytes(type));
  if (st == TM_OK) st = check_cache(num_pages, value_page_stride, kv_heads, "value_cache", elem_bytes(type));
  if (st == TM_OK) st = check_stride(query_stride, heads * kHeadDim, rows, "query");
  if (st == TM_OK) st = check_stride(key_stride, kv_heads * kHeadDim, rows, "key");
  if (st == TM_OK) st = check_stride(value_stride, kv_heads * kHeadDim, rows, "value");
  if (st == TM_OK) st = check_stride(query_out_stride, heads * kHeadDim, rows, "query_out");
  if (st != TM_OK || rows == 0) return st;
  st = check_aligned({query, key, value, query_out, key_cache, value_cache});
  if (st == TM_OK) st = check_element(positions, 8);
  if (st == TM_OK) st = check_element(slot_mapping, 8);
  if (st == TM_OK) st = check_element(frequencies, 8);
  if (st != TM_OK) return st;
  const Rows out{query_out, query_out_stride * 2, heads * kHeadBytes, rows, "query_out"};
  const Rows q{query, query_stride * 2, heads * kHeadBytes, rows, "query"};
  const Rows k{key, key_stride * 2, kv_heads * kHeadBytes, rows, "key"};
  const Rows v{value, value_stride * 2, kv_heads * kHeadBytes, rows, "value"};
  if (!same(q, out) && overlap(out, q)) return refuse_overlap("query_out", "query");
  for (const Rows& other : {k, v}) {
    if (overlap(out, other)) return refuse_overlap("query_out", other.name);
  }
  const Range written[] = {
      out.range(),
      {key_cache, cache_bytes(num_pages, key_page_stride, kv_heads, elem_bytes(type)), "key_cache"},
      {value_cache, cache_bytes(num_pages, value_page_stride, kv_heads, elem_bytes(type)), "value_cache"}};
  const Range small[] = {{positions, rows * 8, "positions"},
                         {slot_mapping, rows * 8, "slot_mapping"},
                         {frequencies, rotary_dim / 2 * 8, "frequencies"},
                         {key_scale, key_scale ? kv_heads * 4 : 0, "key_scale"},
                         {value_scale, value_scale ? kv_heads * 4 : 0, "value_scale"}};
  for (const Range& cache : {written[1], written[2]}) {
    for (const Rows& rows_read : {q, k, v}) {
      if (tmx::overlap(cache, rows_read.range())) return refuse_overlap(cache.name, rows_read.name);
    }
  }
  const bool interleaved_pages = key_page_stride == value_page_stride && num_pages > 1;
  const Rows key_pages{key_cache, key_page_stride * elem_bytes(type), kPageSize * kv_heads * kHeadDim * elem_bytes(type),
                       num_pages, "key_cache"};
  const Rows value_pages{value_cache, value_page_stride * elem_bytes(type),
                         kPageSize * kv_heads * kHeadDim * elem_bytes(type), num_pages, "value_cache"};
  if (interleaved_pages ? overlap(key_pages, value_pages) : tmx::overlap(written[1], written[2])) {
    return refuse_overlap("key_cache", "value_cache");
  }
  for (const Range& w : written) {
    const Range one[] = {w};
    st = check_overlap(one, small);
    if (st != TM_OK) return st;
  }
  for (const Range& cache : {written[1], written[2]}) {
    if (tmx::overlap(written[0], cache)) return refuse_overlap("query_out", cache.name);
  }
  RotateParams p{};
  p.query = static_cast<const uint16_t*>(query);
  p.key = static_cast<const uint16_t*>(key);
  p.value = static_cast<const uint16_t*>(value);
  p.query_out = static_cast<uint16_t*>(query_out);
  p.query_stride = query_stride;
  p.key_stride = key_stride;
  p.value_stride = value_stride;
  p.out_stride = query_out_stride;
  p.positions = positions;
  p.slots = slot_mapping;
  p.frequencies = frequencies;
  p.key_cache = static_cast<char*>(key_cache);
  p.value_cache = static_cast<char*>(value_cache);
  p.key_page_stride = key_page_stride * elem_bytes(type);
  p.value_page_stride = value_page_stride * elem_bytes(type);
  p.key_scale = key_scale;
  p.value_scale = value_scale;
  p.num_slots = num_pages * kPageSize;
  p.rows = (int)rows;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.rotary_dim = (int)rotary_dim;
  p.magnitude = magnitude;
  return launched(launch_rotate(p, interleaved != 0, dtype == TM_FP16, type, static_cast<hipStream_t>(stream)));
}

int64_t tm_cached_attention_workspace_size(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                           int64_t table_cols, int64_t window, int64_t sinks) {
  report(TM_OK, "%s", "");
  if (check_cached(batch, rows, heads, kv_heads, table_cols, window, sinks) != TM_OK) return -1;
  if (batch == 0 || rows == 0) return 0;
  // What either cache type needs, of those whose call is not refused.
  int64_t bytes = -1;
  for (const CacheType type : {CacheType::kSame, CacheType::kE4m3}) {
    const CachedPlan plan = cached_plan(type, batch, rows, heads, kv_heads, table_cols, window, sinks);
    if (check_tiles(plan.tiles) == TM_OK) bytes = std::max(bytes, plan.workspace_bytes);
  }
  if (bytes >= 0) report(TM_OK, "%s", "");
  return bytes;
}

int tm_cached_attention(const void* query, int64_t query_stride, const void* key_cache, int64_t key_page_stride,
                        const void* value_cache, int64_t value_page_stride, const float* key_scale,
                        const float* value_scale, const int32_t* block_table, int64_t table_stride,
                        const int32_t* seq_lens, void* out, int64_t batch, int64_t rows, int64_t heads,
                        int64_t kv_heads, int64_t table_cols, int64_t num_pages, int64_t window, int64_t sinks,
                        float scale, int dtype, int cache_dtype, void* workspace, int64_t workspace_bytes,
                        void* stream) {
  int st = check_dtype(dtype);
  if (st == TM_OK) st = check_cached(batch, rows, heads, kv_heads, table_cols, window, sinks);
  if (st == TM_OK) st = check_table(table_cols, table_stride, batch);
  CacheType type;
  if (st == TM_OK) st = check_cache_type(dtype, cache_dtype, key_scale, value_scale, &type);
  if (st == TM_OK) st = check_cache(num_pages, key_page_stride, kv_heads, "key_cache", elem_bytes(type));
  if (st == TM_OK) st = check_cache(num_pages, value_page_stride, kv_heads, "value_cache", elem_bytes(type));
  if (st == TM_OK) st = check_stride(query_stride, heads * kHeadDim, batch * rows, "query");
  if (st == TM_OK) st = check_scale(scale);
  if (st != TM_OK || batch == 0 || rows == 0) return st;
  st = check_aligned({query, key_cache, value_cache, out});
  if (st == TM_OK) st = check_element(block_table, 4);
  if (st == TM_OK) st = check_element(seq_lens, 4);
  if (st != TM_OK) return st;
  const CachedPlan plan = cached_plan(type, batch, rows, heads, kv_heads, table_cols, window, sinks);
  st = check_tiles(plan.tiles);
  if (st == TM_OK) st = check_workspace(workspace, workspace_bytes, plan.workspace_bytes);
  if (st != TM_OK) return st;
  const Range written[] = {{out, batch * rows * heads * kHeadBytes, "out"},
                           {workspace, plan.workspace_bytes, "workspace"}};
  const Range read[] = {
      {query, rows_bytes(batch * rows, query_stride, heads * kHeadDim), "query"},
      {key_cache, cache_bytes(num_pages, key_page_stride, kv_heads, elem_bytes(type)), "key_cache"},
      {value_cache, cache_bytes(num_pages, value_page_stride, kv_heads, elem_bytes(type)), "value_cache"},
      {key_scale, key_scale ? kv_heads * 4 : 0, "key_scale"},
      {value_scale, value_scale ? kv_heads * 4 : 0, "value_scale"},
      {block_table, table_bytes(batch, table_stride, table_cols), "block_table"},
      {seq_lens, batch * 4, "seq_lens"}};
  st = check_overlap(written, read);
  if (st != TM_OK) return st;
  CachedParams p{};
  p.query = static_cast<const uint16_t*>(query);
  p.query_stride = query_stride;
  p.key_cache = static_cast<const char*>(key_cache);
  p.value_cache = static_cast<const char*>(value_cache);
  p.key_page_stride = key_page_stride * elem_bytes(type);
  p.value_page_stride = value_page_stride * elem_bytes(type);
  p.key_scale = key_scale;
  p.value_scale = value_scale;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.seq_lens = seq_lens;
  p.out = static_cast<uint16_t*>(out);
  if (plan.workspace_bytes > 0) {
    p.counters = static_cast<unsigned long long*>(workspace);
    p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
    p.epoch = workspace_tag(workspace);
  }
  p.table_cols = (int)table_cols;
  p.batch = (int)batch;
  p.rows = (int)rows;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads);
  p.num_pages = (int)num_pages;
  p.window = (int)(window >= INT32_MAX ? -1 : window);  // past every position: all keys
  p.sinks = (int)std::min<int64_t>(sinks, table_cols * kPageSize);
  p.row_shift = plan.row_shift;
  p.key_shift = plan.key_shift;
  p.part_tokens = plan.part_tokens;
  p.row_parts = plan.row_parts;
  p.full_parts = plan.full_parts;
  p.splits = plan.splits;
  p.full_shares = plan.full_shares;
  p.min_tiles = plan.min_tiles;
  p.halvings = plan.halvings;
  p.workgroups = plan.workgroups;
  p.scale_log2 = scale * 1.4426950408889634f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return launched(plan.row_parts > 0 ? launch_cached_chunks(p, plan.shape.rows, dtype == TM_FP16, type, s)
                                     : launch_cached_attention(p, plan.shape, dtype == TM_FP16, type, s));
}

}  // extern "C"
