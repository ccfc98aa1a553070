// Attention of groups of query rows over lists of KV pages, for MI355X
// (gfx950): attention over selected pages, and over draft trees.
//
// Work
// ----
// A group is the query rows that read the same K/V: (request, KV head) with
// all heads of the GQA group, and the rows of one selection block (32 tokens)
// or of one draft tree; rows are numbered token * G + head of the group, and a
// group of more rows than a workgroup's shape holds is cut into several.  A
// unit is one page (128 keys) of one group; a tree's own nodes are its group's
// last unit.  The units of all groups, in a row, are dealt to the workgroups
// in equal contiguous runs, so every workgroup streams the same number of pages
// whatever the lengths in the batch are, and the grid does not depend on them:
// lengths are read on the device, a captured call can be replayed with others.
// A group whose units lie in one workgroup is written by it.  Otherwise each
// of its workgroups leaves an fp32 partial (O, row max, row sum) in the
// workspace and counts its arrival, and the one that arrives last merges them
// in order (the same sums whichever is last) and writes the rows.
//
// A workgroup is four waves = RW row parts x KW = 4 / RW key parts; a wave owns
// 16 NT rows.  Each page goes HBM -> LDS by DMA, 32 KB of K and 32 KB of V, one
// page ahead of the one being read (two K and two V slots, distinct objects,
// so that the compiler sees that the prefetch does not alias the reads): 64 KB
// in flight per CU.  With one row part each wave loads and reads its own 32
// keys of every page and no barrier is needed; with more the page is shared.
//
// Contractions (per wave, 32 keys x 16 rows, v_mfma_f32_16x16x32)
//   S^T (keys x rows) = K Q^T     A = K rows from LDS, B = Q in registers
//   O^T (dims x rows) += V^T P^T  A = V by ds_read_b64_tr_b16, B = P
// Lane l holds row l % 16; accumulator element i of the two 16-key halves is key
// 4 (l / 16) + i (+ 16).  These eight keys are the lane's k-slots of the PV
// operand, so P goes from the accumulators to the operand in registers.
//
// Numerics: scores, row max, row sum and O in fp32, exponentials as exp2 of
// scores in units of log2(e); P is rounded to the input type for the PV
// product (the row sum adds the unrounded values), the output once.  A row
// without keys gives zeros.  K and V rows past a page's valid keys are never
// read from memory (the DMA's range ends there and gives zeros).  In tiles where some row masks a
// key, V entries that are not finite are kept out of the product and added
// only to rows that attend them, so that what a row does not attend cannot
// reach it.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_device.h"
#include "trianglemix_pages.h"

namespace tmx {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short i16x8_t __attribute__((ext_vector_type(8)));

struct Bf16 {
  typedef __bf16 elem;
  typedef bf16x8_t vec;
  static constexpr unsigned kExp = 0x7f80;  // exponent bits: all set in infinities and NaNs
  static constexpr short kOne = 0x3f80;
  static __device__ __forceinline__ f32x4_t mfma(i16x8_t a, i16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};
struct Fp16 {
  typedef _Float16 elem;
  typedef f16x8_t vec;
  static constexpr unsigned kExp = 0x7c00;
  static constexpr short kOne = 0x3c00;
  static __device__ __forceinline__ f32x4_t mfma(i16x8_t a, i16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kSlotBytes = kPageSize * kRowBytes;  // 32 KB: K or V of one page
constexpr int kDmaPerWave = 2 * 8;                 // 1 KB instructions of a wave per page: its 32 keys of K and V
constexpr int kCpolAgent = 16;                     // sc1: seen by every XCD

// Max / sum over the four lanes that hold one row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float row_max(float x) {
  x = half_max(x);
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float x) {
  x = half_sum(x);
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The 16 bytes of K at chunk c of key row r sit in slot c ^ (r % 16) of the
// row, those of V in slot c ^ (4 (r % 4)): both operand reads are free of bank
// conflicts.
__device__ __forceinline__ i16x8_t v_operand16(const char* vt, int off) {
  const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(vt + off));
  const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) i16x4_t*)(vt + off + 16 * kRowBytes));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A value that every lane holds alike, in scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

// A run of consecutive units of one group.
struct Segment {
  int request, kv_head;
  int row0;        // first query row (token) of the group in query / out
  int tokens;      // its tokens
  int row_base;    // first of its rows (token * group + head) this workgroup holds
  int pos0;        // position of token row0 (selected pages)
  int held;        // first tokens without a row (negative positions)
  int lo, hi;      // pages
  int units;       // pages of the whole group
  int64_t first;   // the group's first unit
};

template <class Type, int NT, int RW, bool kTree>
__global__ void __launch_bounds__(kThreads, 1) rows_attention_kernel(const RowsParams p) {
  constexpr int KW = kWaves / RW;
  constexpr int kWaveRows = 16 * NT;
  constexpr int kRows = kWaveRows * RW;
  typedef typename Type::elem elem;

  __shared__ __attribute__((aligned(1024))) char k_lds0[kSlotBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds0[kSlotBytes];
  __shared__ __attribute__((aligned(1024))) char k_lds1[kSlotBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds1[kSlotBytes];
  __shared__ float s_max[kWaves][kWaveRows], s_sum[kWaves][kWaveRows];
  // trees: running unit counts of the requests; selected pages: the list of one
  // selection, and the set it is made from
  __shared__ int64_t s_units[kTree ? kMaxBatch : 1];
  __shared__ unsigned s_set[kTree ? 1 : kMaxTableCols / 32];
  __shared__ int s_list[kTree ? 1 : kMaxSelected];
  __shared__ int s_count[kWaves];
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15;   // row of the wave's 16-row tile
  const int quad = lane >> 4;
  const int rw = wave % RW, kw = wave / RW;
  const int G = p.group;

  // Workgroups are dispatched round-robin over the 8 XCDs: neighbouring runs of
  // units, which share K/V pages where selections overlap, go to one XCD.
  const int run = (int)((blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8);

  // ---- the plan: units, and this workgroup's run of them ----
  auto tree_of = [&](int b, int& row0, int& tokens, int& pages) {
    const int at = p.tree_offsets[b], end = p.tree_offsets[b + 1];
    row0 = min(max(at, 0), p.total_rows);
    tokens = min(min(max(end, row0), p.total_rows) - row0, kMaxTreeNodes);
    const int context = min(max(p.lens[b], 0), p.table_cols * kPageSize);
    pages = (context + kPageSize - 1) / kPageSize;
  };
  int64_t total;
  if constexpr (kTree) {
    // four consecutive requests a thread, prefix sums over the workgroup
    int64_t mine[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = 4 * tid + i;
      mine[i] = 0;
      if (b < p.batch) {
        int row0, tokens, pages;
        tree_of(b, row0, tokens, pages);
        mine[i] = (int64_t)p.kv_heads * ((tokens * G + kRows - 1) / kRows) * (pages + 1);
      }
      sum += mine[i];
    }
    int64_t* scan = reinterpret_cast<int64_t*>(k_lds0);
    scan[tid] = sum;
    __syncthreads();
    for (int d = 1; d < kThreads; d <<= 1) {
      const int64_t add = tid >= d ? scan[tid - d] : 0;
      __syncthreads();
      scan[tid] += add;
      __syncthreads();
    }
    int64_t upto = scan[tid] - sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      upto += mine[i];
      s_units[4 * tid + i] = upto;
    }
    __syncthreads();
    total = uniform64(s_units[p.batch - 1]);
    __syncthreads();
  } else {
    const int row_parts = (min(p.rows, kSelectRows) * G + kRows - 1) / kRows;
    total = (int64_t)p.batch * p.blocks * p.kv_heads * row_parts * p.count;
  }
  const int64_t per_run = max((int64_t)p.min_units, (total + p.workgroups - 1) / p.workgroups);
  int64_t unit = run * per_run;
  const int64_t unit_end = min(total, unit + per_run);

  const int page_row_bytes = p.kv_heads * kRowBytes;

  while (unit < unit_end) {
    Segment g;
    bool draft_last = false;
    int context = 0;  // trees: keys of the cache; selected pages: unused
    int row_parts;
    if constexpr (kTree) {
      int lo = 0, hi = p.batch - 1;  // the request whose running count first passes `unit`
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (s_units[mid] > unit) hi = mid; else lo = mid + 1;
      }
      g.request = __builtin_amdgcn_readfirstlane(lo);
      int pages;
      tree_of(g.request, g.row0, g.tokens, pages);
      g.units = pages + 1;
      row_parts = (g.tokens * G + kRows - 1) / kRows;
      const int64_t before = g.request > 0 ? uniform64(s_units[g.request - 1]) : 0;
      const int local = (int)((unit - before) / g.units);
      g.kv_head = local / row_parts;
      g.row_base = (local % row_parts) * kRows;
      g.first = before + (int64_t)local * g.units;
      context = min(max(p.lens[g.request], 0), p.table_cols * kPageSize);
      g.pos0 = 0;
      g.held = 0;
    } else {
      row_parts = (min(p.rows, kSelectRows) * G + kRows - 1) / kRows;
      g.units = p.count;
      int64_t id = unit / p.count;
      g.first = id * p.count;
      // KV head outermost: the blocks of one head share its pages
      g.row_base = (int)(id % row_parts) * kRows;
      id /= row_parts;
      const int blk = (int)(id % p.blocks);
      id /= p.blocks;
      g.request = (int)(id % p.batch);
      g.kv_head = (int)(id / p.batch);
      g.row0 = g.request * p.rows + blk * kSelectRows;
      g.tokens = min(kSelectRows, p.rows - blk * kSelectRows);
      g.pos0 = max(p.lens[g.request], 0) - p.rows + blk * kSelectRows;
      g.held = max(0, -g.pos0);
    }
    g.lo = (int)(unit - g.first);
    g.hi = (int)(min(unit_end, g.first + g.units) - g.first);
    const bool whole = g.lo == 0 && g.hi == g.units;
    const int valid_rows = min(kRows, g.tokens * G - g.row_base);  // may be <= 0 for a block's last row part

    // ---- the pages: list index i -> logical page; physical page or -1 ----
    const int32_t* const table = p.block_table + g.request * p.table_stride;
    int list_len;        // pages of the list
    bool in_lds = false;  // the list is in s_list, else (selected) in entry / (tree) the index itself
    int entry = 0;
    if constexpr (kTree) {
      list_len = g.units - 1;
    } else {
      const int last = g.pos0 + g.tokens - 1;
      const int possible = last < 0 ? 0 : min(p.table_cols, last / kPageSize + 1);
      const int32_t* const chosen =
          p.selected + ((int64_t)(g.row0 - g.request * p.rows) / kSelectRows + (int64_t)g.request * p.blocks) *
                           p.kv_heads * p.count + (int64_t)g.kv_head * p.count;
      bool sorted = false;
      if (p.count <= 64) {
        // As select_pages leaves it: ascending, what is no page of the block behind.
        entry = lane < p.count ? chosen[lane] : -1;
        const bool ok = entry >= 0 && entry < possible;
        const int before = __shfl_up(ok ? entry : 0x7fffffff, 1);
        sorted = !__any(ok && lane > 0 && before >= entry);
        list_len = __popcll(__ballot(ok));
      }
      if (!sorted) {
        // Any order, entries repeated or out of range: through the set of pages.
        const int words = (possible + 31) / 32;
        __syncthreads();
        for (int i = tid; i < words; i += kThreads) s_set[i] = 0;
        __syncthreads();
        for (int i = tid; i < p.count; i += kThreads) {
          const int e = chosen[i];
          if (e >= 0 && e < possible) atomicOr(&s_set[e >> 5], 1u << (e & 31));
        }
        __syncthreads();
        int base = 0;
        for (int w0 = 0; w0 < words; w0 += kThreads) {
          unsigned bits = w0 + tid < words ? s_set[w0 + tid] : 0;
          const int n = __popc(bits);
          int upto = n;
          for (int d = 1; d < 64; d <<= 1) {
            const int add = __shfl_up(upto, d);
            if (lane >= d) upto += add;
          }
          if (lane == 63) s_count[wave] = upto;
          __syncthreads();
          int at = base + upto - n;
          for (int w = 0; w < wave; ++w) at += s_count[w];
          base += s_count[0] + s_count[1] + s_count[2] + s_count[3];
          while (bits) {  // at most count entries in all
            s_list[at++] = 32 * (w0 + tid) + __ffs(bits) - 1;
            bits &= bits - 1;
          }
          __syncthreads();
        }
        list_len = base;
        in_lds = true;
      }
    }
    list_len = __builtin_amdgcn_readfirstlane(list_len);
    // Pages 64 t .. 64 t + 63 of the list, one a lane.
    int logical64 = 0, phys64 = 0;
    auto load_pages = [&](int t) {
      const int i = 64 * t + lane;
      if constexpr (kTree) {
        logical64 = i;
      } else {
        logical64 = !in_lds ? entry : i < list_len ? s_list[i] : 0;
      }
      phys64 = i < list_len ? table[logical64] : -1;
      if (phys64 >= p.num_pages) phys64 = -1;
    };
    const int last_page = kTree ? g.hi : min(g.hi, list_len);  // pages g.lo .. last_page - 1 are read

    // ---- Q ----
    i16x8_t q[NT][4];
    int row_pos[NT];  // selected pages: the row's position; trees: unused
    uint64_t row_mask[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = rw * kWaveRows + 16 * n + col;
      const int t = (g.row_base + r) / G;
      const int h = g.row_base + r - t * G;
      const bool ok = r < valid_rows;
      row_pos[n] = ok ? g.pos0 + t : -1;
      row_mask[n] = 0;
      if constexpr (kTree) {
        if (ok) row_mask[n] = (uint64_t)p.tree_mask[g.row0 + t];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        i16x8_t x = {};
        if (ok) {
          x = *reinterpret_cast<const i16x8_t*>(p.query + (int64_t)(g.row0 + t) * p.query_stride +
                                                (int64_t)(g.kv_head * G + h) * kHeadDim + 32 * c + 8 * quad);
        }
        q[n][c] = x;
      }
    }

    float m_run[NT], l_run[NT];
    f32x4_t o[8][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m_run[n] = -INFINITY;
      l_run[n] = 0.0f;
#pragma unroll
      for (int m = 0; m < 8; ++m) o[m][n] = f32x4_t{};
    }

    // ---- DMA of page i into a slot pair: this wave's 32 keys ----
    auto issue = [&](int i, char* k_slot_base, char* v_slot_base) {
      const char *kb, *vb;
      int k_rb = page_row_bytes, v_rb = page_row_bytes, valid;
      if (kTree && i == g.units - 1) {
        kb = p.draft_key + (int64_t)g.row0 * p.draft_key_stride;
        vb = p.draft_value + (int64_t)g.row0 * p.draft_value_stride;
        k_rb = (int)p.draft_key_stride;
        v_rb = (int)p.draft_value_stride;
        valid = g.tokens;
      } else {
        const int phys = __builtin_amdgcn_readlane(phys64, i & 63);
        const int at = max(phys, 0);
        kb = p.key_cache + at * p.key_page_stride;
        vb = p.value_cache + at * p.value_page_stride;
        if constexpr (kTree) {
          valid = min(kPageSize, context - i * kPageSize);
        } else {
          const int logical = __builtin_amdgcn_readlane(logical64, i & 63);
          valid = min(kPageSize, g.pos0 + g.tokens - logical * kPageSize);
        }
        if (phys < 0) valid = 0;
      }
      kb += g.kv_head * kRowBytes;
      vb += g.kv_head * kRowBytes;
      const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
          (void*)kb, (short)0, valid > 0 ? (valid - 1) * k_rb + kRowBytes : 0, kBufferFlags);
      const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
          (void*)vb, (short)0, valid > 0 ? (valid - 1) * v_rb + kRowBytes : 0, kBufferFlags);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 32 * wave + 4 * j + quad;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, TM_LDS(k_slot_base + wave * kTileBytes + j * 1024), 16,
                                                 (unsigned)(row * k_rb + 16 * k_slot(row, col)), 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 32 * wave + 4 * j + quad;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, TM_LDS(v_slot_base + wave * kTileBytes + j * 1024), 16,
                                                 (unsigned)(row * v_rb + 16 * v_slot(row, col)), 0, 0, 0);
      }
    };

    const int v_key = 4 * quad + (col >> 2);
    const float c2 = p.scale_log2;

    // One tile of 32 keys, the first at offset t32 of its page.  thr(n): the
    // last key offset in the page that row n attends; draft: by mask bits.
    auto tile = [&](const char* kt, const char* vt, int t32, bool draft, bool masked, const int* thr) {
      f32x4_t s[2][NT];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[u][n] = f32x4_t{};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = 16 * u + col;
          const i16x8_t a = *reinterpret_cast<const i16x8_t*>(kt + row * kRowBytes + 16 * k_slot(row, 4 * c + quad));
#pragma unroll
          for (int n = 0; n < NT; ++n) s[u][n] = Type::mfma(a, q[n][c], s[u][n]);
        }
      }
      if (masked) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = t32 + 16 * u + 4 * quad + i;
              bool seen = key <= thr[n];
              if (kTree && draft) seen = seen && ((row_mask[n] >> (key & 63)) & 1) != 0;
              s[u][n][i] = seen ? s[u][n][i] : -INFINITY;
            }
          }
        }
      }
      i16x8_t pb[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(s[0][n][i], s[1][n][i]));
        top = row_max(top) * c2;
        if (__any(top > m_run[n] + kLazyRescale)) {
          const float m_new = fmaxf(m_run[n], top);
          const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run[n] - m_new);
          l_run[n] *= alpha;
#pragma unroll
          for (int m = 0; m < 8; ++m) o[m][n] *= alpha;
          m_run[n] = m_new;
        }
        const float shift = m_run[n] == -INFINITY ? 0.0f : m_run[n];
        typename Type::vec pv;
        float add = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][n][i], c2, -shift));
            add += e;
            pv[4 * u + i] = (elem)e;
          }
        }
        l_run[n] += add;
        pb[n] = __builtin_bit_cast(i16x8_t, pv);
      }
      // V^T of dims 16 m .. 16 m + 15
      auto v_at = [&](int m) {
        const int d = 16 * m + 4 * (col & 3);
        return v_operand16(vt, v_key * kRowBytes + 16 * v_slot(v_key, d >> 3) + 2 * (d & 7));
      };
      if (masked) {
        bool bad = false;
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          const i16x8_t a = v_at(m);
#pragma unroll
          for (int e = 0; e < 8; ++e) bad |= ((unsigned)a[e] & Type::kExp) == Type::kExp;
        }
        if (__any(bad)) {
#pragma unroll
          for (int m = 0; m < 8; ++m) {
            const i16x8_t a = v_at(m);
            i16x8_t finite, plus, minus, nan;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const unsigned bits = (unsigned)a[e] & 0x7fffu;
              finite[e] = bits < Type::kExp ? a[e] : (short)0;
              plus[e] = bits == Type::kExp && a[e] >= 0 ? Type::kOne : (short)0;
              minus[e] = bits == Type::kExp && a[e] < 0 ? Type::kOne : (short)0;
              nan[e] = bits > Type::kExp ? Type::kOne : (short)0;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              o[m][n] = Type::mfma(finite, pb[n], o[m][n]);
              const f32x4_t has_plus = Type::mfma(plus, pb[n], f32x4_t{});
              const f32x4_t has_minus = Type::mfma(minus, pb[n], f32x4_t{});
              const f32x4_t has_nan = Type::mfma(nan, pb[n], f32x4_t{});
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (has_nan[i] > 0.0f || (has_plus[i] > 0.0f && has_minus[i] > 0.0f)) {
                  o[m][n][i] = __uint_as_float(0x7fc00000u);
                } else if (has_plus[i] > 0.0f) {
                  o[m][n][i] += __uint_as_float(0x7f800000u);
                } else if (has_minus[i] > 0.0f) {
                  o[m][n][i] += __uint_as_float(0xff800000u);
                }
              }
            }
          }
          return;
        }
      }
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const i16x8_t a = v_at(m);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[m][n] = Type::mfma(a, pb[n], o[m][n]);
      }
    };

    // Page i from its slots.
    auto page = [&](int i, const char* ks, const char* vs) {
      int thr[NT];
      int last_seen, first_hidden;  // the last key offset any row attends, the first that some row does not
      bool draft = false;
      if (kTree && i == g.units - 1) {
        draft = true;
        last_seen = g.tokens - 1;
        first_hidden = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) thr[n] = last_seen;
      } else {
        const bool bad = __builtin_amdgcn_readlane(phys64, i & 63) < 0;
        if constexpr (kTree) {
          last_seen = bad ? -1 : min(kPageSize, context - i * kPageSize) - 1;
          first_hidden = last_seen + 1;
#pragma unroll
          for (int n = 0; n < NT; ++n) thr[n] = last_seen;
        } else {
          const int key0 = __builtin_amdgcn_readlane(logical64, i & 63) * kPageSize;
          last_seen = bad ? -1 : g.pos0 + g.tokens - 1 - key0;
          first_hidden = g.pos0 + 1 - key0;
#pragma unroll
          for (int n = 0; n < NT; ++n) thr[n] = row_pos[n] - key0;
        }
      }
      const int tiles = min(4, (last_seen + 32) >> 5);  // tiles with an attended key
      for (int t = kw; t < tiles; t += KW) {
        tile(ks + t * kTileBytes, vs + t * kTileBytes, 32 * t, draft, 32 * t + 31 >= first_hidden, thr);
      }
    };

    // Page i in the slots (ka, va), page i + 1 on its way into (kb, vb).
    int table_block = g.lo >> 6;
    load_pages(table_block);
    auto step = [&](int i, char* ka, char* va, char* kb, char* vb) {
      if constexpr (RW > 1) __syncthreads();  // every wave has read (kb, vb)
      if (i + 1 < last_page) {
        // the page numbers of page i + 1; page i's are needed below
        const int keep_phys = __builtin_amdgcn_readlane(phys64, i & 63);
        const int keep_logical = __builtin_amdgcn_readlane(logical64, i & 63);
        if (((i + 1) & 63) == 0) {
          load_pages((i + 1) >> 6);
          issue(i + 1, kb, vb);
          // lane 63 of the new block is not needed before page i + 64
          if (lane == 63) {
            phys64 = keep_phys;
            logical64 = keep_logical;
          }
        } else {
          if ((i & 63) == 0 && i > g.lo) load_pages(i >> 6);
          issue(i + 1, kb, vb);
        }
        wait_dma_but<kDmaPerWave>();
      } else {
        wait_dma();
      }
      if constexpr (RW > 1) {
        __syncthreads();
      } else {
        asm volatile("" ::: "memory");
      }
      page(i, ka, va);
    };
    if (g.lo < last_page) {
      if constexpr (RW > 1) __syncthreads();
      issue(g.lo, k_lds0, v_lds0);
      int i = g.lo;
      for (; i + 1 < last_page; i += 2) {
        step(i, k_lds0, v_lds0, k_lds1, v_lds1);
        step(i + 1, k_lds1, v_lds1, k_lds0, v_lds0);
      }
      if (i < last_page) step(i, k_lds0, v_lds0, k_lds1, v_lds1);
    }

    // ---- the key parts' sums through LDS; wave w's O in slot w ----
    __syncthreads();
    char* const own = wave == 0 ? k_lds0 : wave == 1 ? v_lds0 : wave == 2 ? k_lds1 : v_lds1;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float l = row_sum(l_run[n]);
      if (quad == 0) {
        s_max[wave][16 * n + col] = m_run[n];
        s_sum[wave][16 * n + col] = l;
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < KW; ++k) top = fmaxf(top, s_max[rw + RW * k][16 * n + col]);
      const float w = m_run[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[n] - top);
      const int row = 16 * n + col;
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const int chunk = (4 * m + quad) ^ col;
        *reinterpret_cast<f32x4_t*>(own + row * (kHeadDim * 4) + 16 * chunk) =
            m_run[n] == -INFINITY ? f32x4_t{} : o[m][n] * w;
      }
    }
    __syncthreads();

    // 16 threads a row, 8 dims each.
    const int r0 = tid >> 4, c8 = tid & 15;
    auto store_row = [&](int r, const float* acc, float l) {
      const int t = (g.row_base + r) / G;
      const int h = g.row_base + r - t * G;
      if (t < g.held) return;  // before the request's first token: no row
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      typename Type::vec y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (elem)(acc[e] * inv);
      *reinterpret_cast<typename Type::vec*>(p.out + ((int64_t)(g.row0 + t) * p.heads + g.kv_head * G + h) * kHeadDim +
                                             8 * c8) = y;
    };
    // the workgroups that share the group, and where their partials lie
    const int first_run = (int)(g.first / per_run);
    const int last_run = (int)((g.first + g.units - 1) / per_run);
    constexpr int kRecord = kRows * (kHeadDim + 2);
    auto record = [&](int r) { return (unsigned)((2 * r + (r == first_run ? 1 : 0)) * (kRecord * 4)); };
    const __amdgpu_buffer_rsrc_t rec = __builtin_amdgcn_make_buffer_rsrc(
        (void*)p.partials, (short)0, whole ? 0 : (int)((unsigned)p.workgroups * 2u * (kRecord * 4u)), kBufferFlags);
    for (int r = r0; r < valid_rows; r += kThreads / 16) {
      const int rp = r / kWaveRows, row = r % kWaveRows;
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < KW; ++k) top = fmaxf(top, s_max[rp + RW * k][row]);
      float l = 0.0f, acc[8] = {};
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const float mk = s_max[rp + RW * k][row];
        l += mk == -INFINITY ? 0.0f : s_sum[rp + RW * k][row] * __builtin_amdgcn_exp2f(mk - top);
        const int w = rp + RW * k;
        const char* src = w == 0 ? k_lds0 : w == 1 ? v_lds0 : w == 2 ? k_lds1 : v_lds1;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const f32x4_t x = *reinterpret_cast<const f32x4_t*>(src + row * (kHeadDim * 4) +
                                                              16 * ((2 * c8 + half) ^ (row & 15)));
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[4 * half + e] += x[e];
        }
      }
      if (whole) {
        store_row(r, acc, l);
      } else {
        const unsigned at = record(run);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const f32x4_t x = {acc[4 * half], acc[4 * half + 1], acc[4 * half + 2], acc[4 * half + 3]};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), rec,
                                                 at + (r * kHeadDim + 8 * c8 + 4 * half) * 4, 0, kCpolAgent);
        }
        if (c8 == 0) {
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(top), rec, at + (kRows * kHeadDim + r) * 4, 0, kCpolAgent);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l), rec, at + (kRows * (kHeadDim + 1) + r) * 4, 0,
                                                kCpolAgent);
        }
      }
    }
    if (!whole) {
      // ---- the workgroup that arrives last merges ----
      // Partials are written through to the level that every XCD sees (sc1) and
      // each wave waits for its own before the arrival is counted.
      wait_dma();
      __syncthreads();
      unsigned long long* const word = p.counters + first_run;
      if (tid == 0) s_last = (int)(count_arrival(word, p.epoch) == (unsigned long long)(last_run - first_run + 1));
      __syncthreads();
      if (s_last) {
        if (tid == 0) __hip_atomic_store(word, p.epoch << kEpochShift, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int r = r0; r < valid_rows; r += kThreads / 16) {
          float top = -INFINITY;
          for (int s = first_run; s <= last_run; ++s) {
            top = fmaxf(top, __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                                 rec, record(s) + (kRows * kHeadDim + r) * 4, 0, kCpolAgent)));
          }
          const float shift = top == -INFINITY ? 0.0f : top;
          float l = 0.0f, acc[8] = {};
#pragma unroll 4
          for (int s = first_run; s <= last_run; ++s) {
            const unsigned at = record(s);
            const float ms = __uint_as_float(
                __builtin_amdgcn_raw_buffer_load_b32(rec, at + (kRows * kHeadDim + r) * 4, 0, kCpolAgent));
            const float ls = __uint_as_float(
                __builtin_amdgcn_raw_buffer_load_b32(rec, at + (kRows * (kHeadDim + 1) + r) * 4, 0, kCpolAgent));
            const float w = __builtin_amdgcn_exp2f(ms - shift);
            l += ls * w;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const f32x4_t x = __builtin_bit_cast(
                  f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                               rec, at + (r * kHeadDim + 8 * c8 + 4 * half) * 4, 0, kCpolAgent));
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[4 * half + e] += ms == -INFINITY ? 0.0f : x[e] * w;
            }
          }
          store_row(r, acc, l);
        }
      }
    }
    unit = g.first + g.hi;
    __syncthreads();
  }
}

template <class Type, bool kTree>
hipError_t launch_shape(const RowsParams& p, int shape_rows, hipStream_t stream) {
  const dim3 grid((unsigned)p.workgroups), block(kThreads);
  switch (shape_rows) {
    case 16: hipLaunchKernelGGL((rows_attention_kernel<Type, 1, 1, kTree>), grid, block, 0, stream, p); break;
    case 32: hipLaunchKernelGGL((rows_attention_kernel<Type, 2, 1, kTree>), grid, block, 0, stream, p); break;
    case 64: hipLaunchKernelGGL((rows_attention_kernel<Type, 4, 1, kTree>), grid, block, 0, stream, p); break;
    case 128: hipLaunchKernelGGL((rows_attention_kernel<Type, 4, 2, kTree>), grid, block, 0, stream, p); break;
    case 256: hipLaunchKernelGGL((rows_attention_kernel<Type, 4, 4, kTree>), grid, block, 0, stream, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rows_attention(const RowsParams& p, int shape_rows, bool fp16, hipStream_t stream) {
  if (p.selected == nullptr) {
    return fp16 ? launch_shape<Fp16, true>(p, shape_rows, stream) : launch_shape<Bf16, true>(p, shape_rows, stream);
  }
  return fp16 ? launch_shape<Fp16, false>(p, shape_rows, stream) : launch_shape<Bf16, false>(p, shape_rows, stream);
}

}  // namespace tmx
