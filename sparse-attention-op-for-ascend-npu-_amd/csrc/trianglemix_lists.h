// Device code that the attention kernels over page lists share
// (trianglemix_rows.hip, trianglemix_blocks.hip): how the work is dealt to the
// workgroups, the list of pages of a group, and the merge of split groups.
//
// A group is the query rows that read the same K/V: (request, KV head) with all
// heads of the GQA group, and the rows of one selection block (32 tokens) or of
// one draft tree; rows are numbered token * G + head of the group, and a group
// of more rows than a workgroup holds is cut into row parts.  A unit is one
// page (128 keys) of one group's row part; a tree's own nodes are its last
// unit.  The units of all groups, in a row, are dealt to the workgroups in equal
// contiguous runs, so every workgroup streams the same number of pages whatever
// the lengths in the batch are, and the grid does not depend on them: lengths
// are read on the device, a captured call can be replayed with others.  A group
// whose units lie in one run is written by its workgroup.  Otherwise each of
// its workgroups leaves an fp32 partial (O, row max, row sum) in the workspace
// and counts its arrival, and the one that arrives last merges them in order
// (the same sums whichever is last) and writes the rows.
#ifndef TRIANGLEMIX_LISTS_H
#define TRIANGLEMIX_LISTS_H

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_device.h"
#include "trianglemix_pages.h"

namespace tmx {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short i16x8_t __attribute__((ext_vector_type(8)));

struct Bf16 {
  typedef __bf16 elem;
  typedef bf16x8_t vec;
  static constexpr unsigned kExp = 0x7f80;  // exponent bits: all set in infinities and NaNs
  static constexpr short kOne = 0x3f80;
  static __device__ __forceinline__ f32x4_t mfma16(i16x8_t a, i16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t mfma32(i16x8_t a, i16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
struct Fp16 {
  typedef _Float16 elem;
  typedef f16x8_t vec;
  static constexpr unsigned kExp = 0x7c00;
  static constexpr short kOne = 0x3c00;
  static __device__ __forceinline__ f32x4_t mfma16(i16x8_t a, i16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t mfma32(i16x8_t a, i16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};

// Of a value's low 16 bits: kind 0 the value where it is finite, else 0; kind
// 1, 2, 3 a one where it is +inf, -inf, NaN, else 0.
template <class Type>
__device__ __forceinline__ unsigned only_kind(unsigned bits, int kind) {
  bits &= 0xffffu;
  const unsigned size = bits & 0x7fffu;
  if (kind == 0) return size < Type::kExp ? bits : 0;
  if (kind == 3) return size > Type::kExp ? (unsigned)Type::kOne : 0;
  return bits == (kind == 1 ? Type::kExp : Type::kExp | 0x8000u) ? (unsigned)Type::kOne : 0;
}

// A row max takes no NaN in: where all scores of a row were NaN it is still -inf,
// but the row sum is NaN, and the row must not pass for one without keys.
__device__ __forceinline__ float row_shift(float max, float sum) {
  return max == -INFINITY && (__float_as_uint(sum) & 0x7fffffffu) != 0 ? 0.0f : max;
}

constexpr int kCpolAgent = 16;  // sc1: written to, read from, the level that every XCD sees

// Workgroups are dispatched round-robin over the 8 XCDs: neighbouring runs of
// units, which share K/V pages where selections overlap, go to one XCD (the
// grid is a multiple of 8).
__device__ __forceinline__ int run_of_workgroup() { return (int)((blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8); }

// Request b's tree: its rows in the batch and the cache's keys, whatever the
// device memory holds.
__device__ __forceinline__ void tree_of(const RowsParams& p, int b, int& row0, int& tokens, int& context) {
  const int at = p.tree_offsets[b], end = p.tree_offsets[b + 1];
  row0 = min(max(at, 0), p.total_rows);
  tokens = min(min(max(end, row0), p.total_rows) - row0, kMaxTreeNodes);
  context = min(max(p.lens[b], 0), p.table_cols * kPageSize);
}

// LDS of the plan and the lists.
template <bool kTree>
struct ListLds;
template <>
struct ListLds<true> {
  int units[kMaxBatch];  // running unit counts of the requests
  int row0[kMaxBatch], size[kMaxBatch];  // their trees (tree_of): first row, context * 128 + tokens
  int64_t scan[16];      // wave totals
};
template <>
struct ListLds<false> {
  unsigned set[kMaxTableCols / 32];  // the pages of one selection, and the list made from them
  int list[kMaxSelected];
  int count[16];
};

// A run of consecutive units of one group.
static_assert(kMaxTreeNodes < 128 && (int64_t)kMaxTableCols * kPageSize * 128 < (int64_t(1) << 31), "a tree's size in 32 bits");
struct Segment {
  int request, kv_head;
  int row0;       // first query row (token) of the group in query / out
  int tokens;     // its tokens
  int row_base;   // first of its rows (token * group + head) this workgroup holds
  int pos0;       // position of token row0 (selected pages)
  int held;       // first tokens without a row (negative positions)
  int context;    // keys of the cache (trees)
  int lo, hi;     // its units
  int units;      // units of the whole group
  int first;      // the group's first unit
};

// r / group for the rows of a group (below 2048): exact, as r * group < 65536.
struct GroupDivider {
  unsigned group, inverse;
  __device__ explicit GroupDivider(int g) : group((unsigned)g), inverse(65536u / (unsigned)g + 1u) {}
  __device__ int token(int row) const { return (int)(((unsigned)row * inverse) >> 16); }
};
static_assert(kMaxTreeNodes * kMaxGroup <= 2048 && kSelectRows * kMaxGroup <= 2048 && 2047 * kMaxGroup < 65536,
              "rows of a group");

// All units (the host keeps them to kMaxUnits), dealt to the runs in equal parts;
// for trees the running counts too.  Every thread of the workgroup calls it.
struct Plan {
  int total, per_run;
};
template <bool kTree, int kRows, int kThreads>
__device__ __forceinline__ Plan plan_units(const RowsParams& p, ListLds<kTree>& lds) {
  if constexpr (kTree) {
    // consecutive requests a thread, prefix sums over the workgroup
    constexpr int kEach = kMaxBatch / kThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t mine[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int b = kEach * tid + i;
      mine[i] = 0;
      if (b < p.batch) {
        int row0, tokens, context;
        tree_of(p, b, row0, tokens, context);
        lds.row0[b] = row0;
        lds.size[b] = context * 128 + tokens;
        mine[i] = (int64_t)(p.kv_heads * ((tokens * p.group + kRows - 1) / kRows)) *
                  ((context + kPageSize - 1) / kPageSize + 1);
      }
      sum += mine[i];
    }
    int64_t upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t add = __shfl_up(upto, d);
      if (lane >= d) upto += add;
    }
    if (lane == 63) lds.scan[wave] = upto;
    __syncthreads();
    upto -= sum;
    for (int w = 0; w < wave; ++w) upto += lds.scan[w];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      upto += mine[i];
      lds.units[kEach * tid + i] = (int)min(upto, (int64_t)kMaxUnits);  // more only with offsets that are none
    }
    __syncthreads();
    const int total = __builtin_amdgcn_readfirstlane(lds.units[p.batch - 1]);
    const int usual = (int)((unsigned)total / (unsigned)(p.kv_heads * p.batch));  // units of a group of one row part
    return Plan{total, max(min_run_units(usual, kRows),
                           (int)((unsigned)(total + p.workgroups - 1) / (unsigned)p.workgroups))};
  } else {
    return Plan{p.total_units, p.per_run};
  }
}

// The segment that begins at `unit` and ends with the group or before unit_end.
template <bool kTree, int kRows>
__device__ __forceinline__ Segment find_segment(const RowsParams& p, const ListLds<kTree>& lds, int unit, int unit_end) {
  Segment g;
  if constexpr (kTree) {
    // the request whose running count first passes `unit` (entries past the batch hold the total)
    int lo = 0;
    for (;; lo += 64) {
      const uint64_t past = __ballot(lds.units[lo + (threadIdx.x & 63)] > unit);
      if (past) {
        lo += __ffsll((unsigned long long)past) - 1;
        break;
      }
    }
    g.request = lo;
    g.row0 = __builtin_amdgcn_readfirstlane(lds.row0[lo]);
    const int size = __builtin_amdgcn_readfirstlane(lds.size[lo]);
    g.tokens = size & 127;
    g.context = size >> 7;
    g.units = (g.context + kPageSize - 1) / kPageSize + 1;
    const int row_parts = (g.tokens * p.group + kRows - 1) / kRows;
    const int before = lo > 0 ? __builtin_amdgcn_readfirstlane(lds.units[lo - 1]) : 0;
    const int local = (int)((unsigned)(unit - before) / (unsigned)g.units);
    g.kv_head = local / row_parts;
    g.row_base = (local % row_parts) * kRows;
    g.first = before + local * g.units;
    g.pos0 = 0;
    g.held = 0;
  } else {
    const unsigned row_parts = (unsigned)(min(p.rows, kSelectRows) * p.group + kRows - 1) / kRows;
    g.units = p.count;
    unsigned id = (unsigned)unit / (unsigned)p.count;
    g.first = (int)(id * (unsigned)p.count);
    // KV head outermost: the blocks of one head share its pages
    g.row_base = (int)(id % row_parts) * kRows;
    id /= row_parts;
    const int blk = (int)(id % (unsigned)p.blocks);
    id /= (unsigned)p.blocks;
    g.request = (int)(id % (unsigned)p.batch);
    g.kv_head = (int)(id / (unsigned)p.batch);
    g.row0 = g.request * p.rows + blk * kSelectRows;
    g.tokens = min(kSelectRows, p.rows - blk * kSelectRows);
    g.pos0 = max(p.lens[g.request], 0) - p.rows + blk * kSelectRows;
    g.held = max(0, -g.pos0);
    g.context = 0;
  }
  g.lo = unit - g.first;
  g.hi = min(unit_end - g.first, g.units);
  return g;
}

// A selection's list in memory, and its first 64 entries, one a lane: loaded
// apart from their use, so that other loads can go along.
__device__ __forceinline__ const int32_t* selection_of(const RowsParams& p, const Segment& g) {
  const int blk = (g.row0 - g.request * p.rows) / kSelectRows;
  return p.selected + (((int64_t)g.request * p.blocks + blk) * p.kv_heads + g.kv_head) * p.count;
}
__device__ __forceinline__ int selection_entry(const RowsParams& p, const int32_t* chosen) {
  const int lane = threadIdx.x & 63;
  return lane < p.count ? chosen[lane] : -1;
}

// The pages of a selection, ascending, each once: in `entry` (page i in lane i;
// in_lds false) or in lds.list.  Returns how many.  Every thread of the
// workgroup calls it, with selection_entry in `entry`.
template <int kThreads>
__device__ __forceinline__ int selected_list(const RowsParams& p, ListLds<false>& lds, const Segment& g,
                                             const int32_t* chosen, int& entry, bool& in_lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int last = g.pos0 + g.tokens - 1;
  const int possible = last < 0 ? 0 : min(p.table_cols, last / kPageSize + 1);
  in_lds = false;
  if (p.count <= 64) {
    // As select_pages leaves it: ascending, what is no page of the block behind.
    const bool ok = entry >= 0 && entry < possible;
    const int before = __shfl_up(ok ? entry : 0x7fffffff, 1);
    if (!__any(ok && lane > 0 && before >= entry)) {
      entry = ok ? entry : 0;
      return __popcll(__ballot(ok));
    }
  }
  // Any order, entries repeated or out of range: through the set of pages.
  in_lds = true;
  const int words = (possible + 31) / 32;
  __syncthreads();
  for (int i = tid; i < words; i += kThreads) lds.set[i] = 0;
  __syncthreads();
  for (int i = tid; i < p.count; i += kThreads) {
    const int e = chosen[i];
    if (e >= 0 && e < possible) atomicOr(&lds.set[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  int base = 0;
  for (int w0 = 0; w0 < words; w0 += kThreads) {
    unsigned bits = w0 + tid < words ? lds.set[w0 + tid] : 0;
    const int n = __popc(bits);
    int upto = n;
    for (int d = 1; d < 64; d <<= 1) {
      const int add = __shfl_up(upto, d);
      if (lane >= d) upto += add;
    }
    if (lane == 63) lds.count[wave] = upto;
    __syncthreads();
    int at = base + upto - n;
    for (int w = 0; w < wave; ++w) at += lds.count[w];
    for (int w = 0; w < kThreads / 64; ++w) base += lds.count[w];
    while (bits) {  // at most count entries in all
      lds.list[at++] = 32 * (w0 + tid) + __ffs(bits) - 1;
      bits &= bits - 1;
    }
    __syncthreads();
  }
  return __builtin_amdgcn_readfirstlane(base);
}

// The runs that share a group, first_run .. last_run, and where run r leaves its
// partial of it: a run has two records, one for a group that began before it
// and one for a group that begins in it and goes on behind it.
struct Shared {
  int first_run, last_run;
  __device__ Shared(const Segment& g, int per_run)
      : first_run((int)((unsigned)g.first / (unsigned)per_run)),
        last_run((int)((unsigned)(g.first + g.units - 1) / (unsigned)per_run)) {}
  __device__ unsigned record(int r, unsigned bytes) const { return (unsigned)(2 * r + (r == first_run ? 1 : 0)) * bytes; }
};

// Counts this workgroup's arrival at its group, whose partial it has stored
// (sc1); true in the workgroup that completes it.  Every thread calls it.
__device__ __forceinline__ bool last_to_arrive(const RowsParams& p, const Shared& shared, int* flag) {
  wait_dma();  // this wave's partial stores have completed
  __syncthreads();
  unsigned long long* const word = p.counters + shared.first_run;
  if (threadIdx.x == 0) {
    *flag = (int)(count_arrival(word, p.epoch) == (unsigned long long)(shared.last_run - shared.first_run + 1));
  }
  __syncthreads();
  const bool last = *flag != 0;
  // The word is left at this launch's tag with a count of zero for the next one.
  if (last && threadIdx.x == 0) {
    __hip_atomic_store(word, p.epoch << kEpochShift, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  return last;
}

}  // namespace tmx

#endif  // TRIANGLEMIX_LISTS_H
