// Attention of small groups of query rows over lists of KV pages, for MI355X
// (gfx950): a decoding step over selected pages, and draft trees.
//
// Work, lists and merge as in trianglemix_lists.h; groups of more rows run in
// trianglemix_blocks.hip.
//
// A workgroup is four waves over the same 16 NT rows; wave w has keys 32 w ..
// 32 w + 31 of every page.  Each page goes HBM -> LDS by DMA, 32 KB of K and
// 32 KB of V, one page ahead of the one being read (two K and two V slots,
// distinct objects, so that the compiler sees that the prefetch does not alias
// the reads): 64 KB in flight per CU.  A wave loads what it reads itself, so
// the page loop has no barrier; the waves' sums meet in LDS behind it.
//
// What bounds it: memory.  24 pages of each KV head for 64 requests of 2000 to
// 16384 tokens (798 MB of K and V) take 138 us, 5.8 TB/s, where a library copy
// of 2 GiB moves 4.9 (read and written).  One
// request's few pages are bound by latency instead (8 us for 64 pages x 8 KV
// heads: launch, lengths, selection, table, page, merge, each waiting for the
// one before).
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
// read from memory (the DMA's range ends there and gives zeros).  In tiles where
// some row masks a key, V entries that are not finite are kept out of the product
// and added only to rows that attend them, so that what a row does not attend
// cannot reach it.  (Elsewhere an infinity whose weight rounds to zero gives NaN.)

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_lists.h"

namespace tmx {
namespace {

constexpr int kSlotBytes = kPageSize * kRowBytes;  // 32 KB: K or V of one page

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

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;

template <class Type, int NT, bool kTree>
__global__ void __launch_bounds__(kThreads, 1) rows_attention_kernel(const RowsParams p) {
  constexpr int kWaveKeys = kPageSize / kWaves;  // keys of a page that a wave loads
  constexpr int kDma = kWaveKeys / 4;            // by this many 1 KB instructions each for K and V
  constexpr int kRows = 16 * NT;
  static_assert(kWaves == 4 && kRows * kHeadDim * 4 <= kSlotBytes, "each wave's O fits a slot");
  typedef typename Type::elem elem;

  __shared__ __attribute__((aligned(1024))) char k_lds0[kSlotBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds0[kSlotBytes];
  __shared__ __attribute__((aligned(1024))) char k_lds1[kSlotBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds1[kSlotBytes];
  __shared__ float s_max[kWaves][kRows], s_sum[kWaves][kRows];
  __shared__ ListLds<kTree> lists;
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15;   // row of the wave's 16-row tile
  const int quad = lane >> 4;
  const int G = p.group;

  const GroupDivider by_group(p.group);
  const int page_row_bytes = p.kv_heads * kRowBytes;

  const Plan plan = plan_units<kTree, kRows, kThreads>(p, lists);
  const int run = run_of_workgroup();
  int unit = min(run, plan.total / plan.per_run + 1) * plan.per_run;
  const int unit_end = min(plan.total, unit + plan.per_run);

  while (unit < unit_end) {
    const Segment g = find_segment<kTree, kRows>(p, lists, unit, unit_end);
    const bool whole = g.lo == 0 && g.hi == g.units;
    const int valid_rows = min(kRows, g.tokens * G - g.row_base);

    // What needs no page number is loaded first: the selection, then Q.
    const int32_t* chosen = nullptr;
    int entry = 0;
    if constexpr (!kTree) {
      chosen = selection_of(p, g);
      entry = selection_entry(p, chosen);
    }
    // ---- Q ----
    i16x8_t q[NT][4];
    int row_pos[NT];  // selected pages: the row's position; trees: unused
    uint64_t row_mask[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 16 * n + col;
      const int t = by_group.token(g.row_base + r);
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

    // ---- the pages: list index i -> logical page; physical page or -1 ----
    const int32_t* const table = p.block_table + g.request * p.table_stride;
    int list_len;  // pages of the list
    bool in_lds = false;
    if constexpr (kTree) list_len = g.units - 1;
    else list_len = selected_list<kThreads>(p, lists, g, chosen, entry, in_lds);
    // Pages 64 t .. 64 t + 63 of the list, one a lane.
    int logical64 = 0, phys64 = 0;
    auto load_pages = [&](int t) {
      const int i = 64 * t + lane;
      if constexpr (kTree) {
        logical64 = i;
      } else {
        logical64 = !in_lds ? entry : i < list_len ? lists.list[i] : 0;
      }
      phys64 = i < list_len ? table[logical64] : -1;
      if (phys64 >= p.num_pages) phys64 = -1;
    };
    const int last_page = kTree ? g.hi : min(g.hi, list_len);  // pages g.lo .. last_page - 1 are read

    float m_run[NT], l_run[NT];
    f32x4_t o[8][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m_run[n] = -INFINITY;
      l_run[n] = 0.0f;
#pragma unroll
      for (int m = 0; m < 8; ++m) o[m][n] = f32x4_t{};
    }

    // ---- DMA of page i into a slot pair: this wave's share of the keys ----
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
          valid = min(kPageSize, g.context - i * kPageSize);
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
      for (int j = 0; j < kDma; ++j) {
        const int row = kWaveKeys * wave + 4 * j + quad;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, TM_LDS(k_slot_base + (wave * kDma + j) * 1024), 16,
                                                 (unsigned)(row * k_rb + 16 * k_slot(row, col)), 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < kDma; ++j) {
        const int row = kWaveKeys * wave + 4 * j + quad;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, TM_LDS(v_slot_base + (wave * kDma + j) * 1024), 16,
                                                 (unsigned)(row * v_rb + 16 * v_slot(row, col)), 0, 0, 0);
      }
    };

    // Swizzled operand addresses differ by an exclusive or alone: K of dims 32 c ..
    // at k_off ^ 64 c, V of dims 16 m .. at v_off ^ 32 m.
    const int k_off = col * kRowBytes + 16 * k_slot(col, quad);
    const int v_key = 4 * quad + (col >> 2), v_dim = 4 * (col & 3);
    const int v_off = v_key * kRowBytes + 16 * v_slot(v_key, v_dim >> 3) + 2 * (v_dim & 7);
    const float c2 = p.scale_log2;

    // One tile of 32 keys, the first at offset t32 of its page.  thr[n]: the last
    // key offset in the page that row n attends; draft: by mask bits too.
    auto tile = [&](const char* kt, const char* vt, int t32, bool draft, bool masked, const int* thr) {
      f32x4_t s[2][NT];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[u][n] = f32x4_t{};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const i16x8_t a = *reinterpret_cast<const i16x8_t*>(kt + 16 * u * kRowBytes + (k_off ^ (64 * c)));
#pragma unroll
          for (int n = 0; n < NT; ++n) s[u][n] = Type::mfma16(a, q[n][c], s[u][n]);
        }
      }
      if (masked) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int limit = thr[n] - t32 - 4 * quad;  // of 16 u + i
          uint32_t bits = ~0u;
          if (kTree && draft) bits = (uint32_t)(row_mask[n] >> (t32 & 63)) >> (4 * quad);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              bool seen = 16 * u + i <= limit;
              if (kTree) seen = seen && (bits & (1u << (16 * u + i))) != 0;
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
      auto v_at = [&](int m) { return v_operand16(vt, v_off ^ (32 * m)); };  // V^T of dims 16 m .. 16 m + 15
      if (masked) {
        typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));
        u16x8_t size = {};
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          size = __builtin_elementwise_max(size, __builtin_bit_cast(u16x8_t, v_at(m) & (short)0x7fff));
        }
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) bad |= size[e] >= Type::kExp;
        if (__builtin_expect(__any(bad) != 0, 0)) {
          // The finite entries, then for each other kind the product of indicators
          // (such an entry; the key attended, whatever its weight rounded to).
          i16x8_t attended[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) attended[n][e] = s[e >> 2][n][e & 3] != -INFINITY ? Type::kOne : 0;
          }
#pragma unroll
          for (int m = 0; m < 8; ++m) {
#pragma unroll
            for (int kind = 0; kind < 4; ++kind) {  // finite, +inf, -inf, NaN
              asm volatile("" ::: "memory");
              u32x4_t a = __builtin_bit_cast(u32x4_t, v_at(m));
              asm volatile("" : "+v"(a));
#pragma unroll
              for (int e = 0; e < 4; ++e) a[e] = only_kind<Type>(a[e], kind) | only_kind<Type>(a[e] >> 16, kind) << 16;
              // opaque: the compiler takes no operand for a NaN; +inf and -inf give one by themselves
              float odd = __uint_as_float(kind == 1 ? 0x7f800000u : kind == 2 ? 0xff800000u : 0x7fc00000u);
              asm volatile("" : "+v"(odd));
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (kind == 0) {
                  o[m][n] = Type::mfma16(__builtin_bit_cast(i16x8_t, a), pb[n], o[m][n]);
                } else {
                  const f32x4_t has = Type::mfma16(__builtin_bit_cast(i16x8_t, a), attended[n], f32x4_t{});
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[m][n][i] += has[i] > 0.0f ? odd : 0.0f;
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
        for (int n = 0; n < NT; ++n) o[m][n] = Type::mfma16(a, pb[n], o[m][n]);
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
          last_seen = bad ? -1 : min(kPageSize, g.context - i * kPageSize) - 1;
          first_hidden = last_seen + 1;
#pragma unroll
          for (int n = 0; n < NT; ++n) thr[n] = last_seen;
        } else {
          const int key0 = __builtin_amdgcn_readlane(logical64, i & 63) * kPageSize;
          last_seen = bad ? -1 : min(g.pos0 + g.tokens - 1 - key0, kPageSize - 1);
          first_hidden = g.pos0 + 1 - key0;
#pragma unroll
          for (int n = 0; n < NT; ++n) thr[n] = row_pos[n] - key0;
        }
      }
      const int tiles = min(4, (last_seen + 32) >> 5);  // tiles with an attended key
      const int t = wave;
      if (t < tiles) tile(ks + t * kTileBytes, vs + t * kTileBytes, 32 * t, draft, 32 * t + 31 >= first_hidden, thr);
    };

    // Page i in the slots (ka, va), page i + 1 on its way into (kb, vb).
    int table_block = g.lo >> 6;
    load_pages(table_block);
    auto step = [&](int i, char* ka, char* va, char* kb, char* vb) {
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
        wait_dma_but<2 * kDma>();
      } else {
        wait_dma();
      }
      asm volatile("" ::: "memory");
      page(i, ka, va);
    };
    if (g.lo < last_page) {
      issue(g.lo, k_lds0, v_lds0);
      int i = g.lo;
      for (; i + 1 < last_page; i += 2) {
        step(i, k_lds0, v_lds0, k_lds1, v_lds1);
        step(i + 1, k_lds1, v_lds1, k_lds0, v_lds0);
      }
      if (i < last_page) step(i, k_lds0, v_lds0, k_lds1, v_lds1);
    }

    // ---- the waves' sums through LDS; each wave's O in a slot ----
    __syncthreads();
    auto o_slot = [&](int w) { return w == 0 ? k_lds0 : w == 1 ? v_lds0 : w == 2 ? k_lds1 : v_lds1; };
    char* const own = o_slot(wave);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float l = row_sum(l_run[n]);
      m_run[n] = row_shift(m_run[n], l);
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
      for (int k = 0; k < kWaves; ++k) top = fmaxf(top, s_max[k][16 * n + col]);
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
      const int t = by_group.token(g.row_base + r);
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
    const Shared shared(g, plan.per_run);
    constexpr int kRecord = kRows * (kHeadDim + 2);
    auto record = [&](int r) { return shared.record(r, kRecord * 4); };
    const __amdgpu_buffer_rsrc_t rec = __builtin_amdgcn_make_buffer_rsrc(
        (void*)p.partials, (short)0, whole ? 0 : (int)((unsigned)p.workgroups * 2u * (kRecord * 4u)), kBufferFlags);
    for (int r = r0; r < valid_rows; r += kThreads / 16) {
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) top = fmaxf(top, s_max[k][r]);
      float l = 0.0f, acc[8] = {};
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float mk = s_max[k][r];
        l += mk == -INFINITY ? 0.0f : s_sum[k][r] * __builtin_amdgcn_exp2f(mk - top);
        const char* src = o_slot(k);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const f32x4_t x = *reinterpret_cast<const f32x4_t*>(src + r * (kHeadDim * 4) +
                                                              16 * ((2 * c8 + half) ^ (r & 15)));
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
      if (last_to_arrive(p, shared, &s_last)) {
        // 16 threads a row again; where the rows leave threads over, they share
        // a row's partials (part pg of `parts` takes every parts-th) and join
        // through LDS.  Four partials' loads are in flight at a time.
        int row_slots = 1;
        while (row_slots < valid_rows && row_slots < kThreads / 16) row_slots *= 2;
        const int parts = kThreads / 16 / row_slots;
        const int pg = r0 / row_slots;
        float* const join = reinterpret_cast<float*>(k_lds0);  // [thread][10]: acc, row max, row sum
        static_assert(kThreads * 10 * 4 <= kSlotBytes, "the joined values fit a slot");
        for (int rb = 0; rb < valid_rows; rb += row_slots) {
          const int r = rb + r0 % row_slots;
          float top = -INFINITY, l = 0.0f, acc[8] = {};
          if (r < valid_rows) {
            for (int s0 = shared.first_run + pg; s0 <= shared.last_run; s0 += 4 * parts) {
              float ms[4], ls[4];
              f32x4_t x[4][2];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                // past the last one its loads fall outside the buffer's range
                const int s = s0 + j * parts;
                const unsigned at = s <= shared.last_run ? record(s) : kOutOfRange;
                ms[j] = __uint_as_float(
                    __builtin_amdgcn_raw_buffer_load_b32(rec, at + (kRows * kHeadDim + r) * 4, 0, kCpolAgent));
                ls[j] = __uint_as_float(
                    __builtin_amdgcn_raw_buffer_load_b32(rec, at + (kRows * (kHeadDim + 1) + r) * 4, 0, kCpolAgent));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  x[j][half] = __builtin_bit_cast(
                      f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                   rec, at + (r * kHeadDim + 8 * c8 + 4 * half) * 4, 0, kCpolAgent));
                }
              }
              float next = top;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (s0 + j * parts > shared.last_run) ms[j] = -INFINITY;
                next = fmaxf(next, ms[j]);
              }
              const float shift = next == -INFINITY ? 0.0f : next;
              const float keep = __builtin_amdgcn_exp2f(top - shift);
              l *= keep;
#pragma unroll
              for (int e = 0; e < 8; ++e) acc[e] *= keep;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float w = __builtin_amdgcn_exp2f(ms[j] - shift);
                l += ls[j] * w;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] += x[j][e >> 2][e & 3] * w;
              }
              top = next;
            }
          }
          if (parts > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) join[tid * 10 + e] = acc[e];
            join[tid * 10 + 8] = top;
            join[tid * 10 + 9] = l;
            __syncthreads();
            if (pg == 0) {
              float all = top;
              for (int k = 1; k < parts; ++k) all = fmaxf(all, join[(tid + k * 16 * row_slots) * 10 + 8]);
              const float shift = all == -INFINITY ? 0.0f : all;
              const float keep = __builtin_amdgcn_exp2f(top - shift);
              l *= keep;
#pragma unroll
              for (int e = 0; e < 8; ++e) acc[e] *= keep;
              for (int k = 1; k < parts; ++k) {
                const float* const from = join + (tid + k * 16 * row_slots) * 10;
                const float w = __builtin_amdgcn_exp2f(from[8] - shift);
                l += from[9] * w;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] += from[e] * w;
              }
            }
          }
          if (pg == 0 && r < valid_rows) store_row(r, acc, l);
        }
      }
    }
    unit = g.first + g.hi;
    __syncthreads();
  }
}

template <class Type, bool kTree>
hipError_t launch_shape(const RowsParams& p, int shape_rows, hipStream_t stream) {
  const dim3 grid((unsigned)p.workgroups);
  switch (shape_rows) {
    case 16: hipLaunchKernelGGL((rows_attention_kernel<Type, 1, kTree>), grid, dim3(256), 0, stream, p); break;
    case 32: hipLaunchKernelGGL((rows_attention_kernel<Type, 2, kTree>), grid, dim3(256), 0, stream, p); break;
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
