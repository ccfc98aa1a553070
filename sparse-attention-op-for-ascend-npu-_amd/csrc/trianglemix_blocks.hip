// Attention of large groups of query rows over lists of KV pages, for MI355X
// (gfx950): selection blocks of a prefill chunk, and large draft trees.  Work,
// lists and merge as in trianglemix_lists.h; groups of few rows run in
// trianglemix_rows.hip.
//
// A workgroup is W waves = W / KP row parts of 32 rows x KP key parts: eight row
// parts for groups of more than 128 rows, four row parts x two key parts for
// smaller ones, or two workgroups of four row parts a CU (when which: the plans
// in trianglemix_pages_capi.cpp).  So a SIMD has two waves, and runs one's softmax
// beside the other's MFMAs.  The loop goes in steps of 32 KP keys, a wave taking
// the 32 of its key part (8 KB of K, 8 KB of V), DMA'd into NS K and NS V slots
// (distinct objects: the compiler sees that the prefetch does not alias the
// reads): K NS steps, V NS - 1 steps ahead of the one in hand.  One half of the
// waves loads K, the other V.  Key parts join through LDS behind the loop.
//
// Software pipeline: iteration i issues the QK^T MFMAs of step i + 1 between
// the exponentials of step i, then the PV MFMAs of step i between the row max of
// step i + 1.  Only steps that every row attends whole run there: lists are
// ascending, so the steps that need a mask (the keys at and after the block's
// first row, the end of a tree's context, the tree itself) are the last ones,
// and run one after the other in a plain loop behind it, with what the pipeline
// leaves over.  There V entries that are not finite are kept out of the product and
// added only to rows that attend them, so that what a row does not attend
// cannot reach it.
//
// Contractions (per wave, v_mfma_f32_32x32x16):
//   S^T (32 keys x 32 rows) = K Q^T, O^T (128 x 32 rows) += V^T P^T,
// lane l holding row l % 32, accumulator element v key 8 (v / 4) + 4 (l / 32) + v % 4;
// the scores of a lane are the k-slots of its PV operand.  Numerics as in
// trianglemix_rows.hip.
//
// What bounds it: with pages that the L2 holds the MFMAs and the exponentials
// beside them, 1028 TFLOP/s over 2048 rows x 128 pages (97 % of the reads hit the
// L2, MFMAs are busy in half the cycles), where a bf16
// library product of 8192^3 reaches 1377; with pages read once, memory: 32 trees
// of up to 32 nodes over 8000 tokens each take 192 us, 5.5 TB/s.  Short lists
// pay for the start (lengths, selection, Q and table before the first step, 7
// us) and the partials of split groups: 512 rows x 16 pages take 34 us.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_lists.h"

namespace tmx {
namespace {

constexpr int kAhead = 3;  // MFMA steps between an LDS operand read and its use
static_assert(kPartialBytes == 128 * (kHeadDim + 4) * 4, "the record of four waves");
template <int J>
struct Index { static constexpr int value = J; };

// Operand reads of a tile.  Swizzled addresses differ by an exclusive or alone:
// one register holds them all.
__device__ __forceinline__ i16x8_t k_operand_of(const char* kt, int k0, int c) {  // dims 16 c .. 16 c + 15
  return *reinterpret_cast<const i16x8_t*>(kt + (k0 ^ (32 * c)));
}
__device__ __forceinline__ i16x8_t v_operand_of(const char* vt, int v0, int k) {  // d-block k % 4, keys 16 (k / 4) ..
  const char* const a = vt + 16 * (k >> 2) * kRowBytes + (v0 ^ (64 * (k & 3)));
  const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)a);
  const i16x4_t hi =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(a + 8 * kRowBytes));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// W waves: W / KP row parts of 32 rows x KP key parts.
template <class Type, int W, int KP, bool kTree>
__global__ void __launch_bounds__(W * 64, 2) blocks_attention_kernel(const RowsParams p) {
  typedef typename Type::elem elem;
  constexpr int kRowParts = W / KP;
  constexpr int NS = W == 4 ? 4 : 6 / KP;  // slots of a step; 64 KB (of two workgroups) or 80 KB in flight per CU
  constexpr int kUnroll = W == 4 ? 4 : 6;  // scores swap buffers every step, slots turn every NS
  constexpr int kStep = KP * kKvTile;  // keys of a step
  constexpr int kSteps = kPageSize / kStep;  // steps of a page
  constexpr int kStepBytes = KP * kTileBytes;
  constexpr int kGroupRows = 32 * kRowParts;
  constexpr int kBlockThreads = 64 * W;
  constexpr int kLoaders = W / 2;                   // waves that share the DMA of K, and of V
  constexpr int kDmaShare = KP * kDmaPerTile / kLoaders;
  constexpr unsigned kRecordBytes = (unsigned)kPartialBytes * (kRowParts / 4);
  static_assert((W == 8 || W == 4) && (KP == 1 || (KP == 2 && W == 8)) && kUnroll % NS == 0 && kUnroll % 2 == 0, "supported shapes");
  __shared__ __attribute__((aligned(1024))) char k_lds0[kStepBytes];
  __shared__ __attribute__((aligned(1024))) char k_lds1[kStepBytes];
  __shared__ __attribute__((aligned(1024))) char k_lds2[kStepBytes];
  __shared__ __attribute__((aligned(1024))) char k_lds3[NS > 3 ? kStepBytes : 16];
  __shared__ __attribute__((aligned(1024))) char k_lds4[NS > 4 ? kStepBytes : 16];
  __shared__ __attribute__((aligned(1024))) char k_lds5[NS > 5 ? kStepBytes : 16];
  __shared__ __attribute__((aligned(1024))) char v_lds0[kStepBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds1[kStepBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds2[kStepBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds3[NS > 3 ? kStepBytes : 16];
  __shared__ __attribute__((aligned(1024))) char v_lds4[NS > 4 ? kStepBytes : 16];
  __shared__ __attribute__((aligned(1024))) char v_lds5[NS > 5 ? kStepBytes : 16];
  __shared__ ListLds<kTree> lists;
  __shared__ int s_last;
  // Slot j, named statically or picked (where nothing is prefetched beside the reads).
  auto k_at = [&](auto j) -> char* {
    constexpr int i = decltype(j)::value % NS;
    return i == 0 ? k_lds0 : i == 1 ? k_lds1 : i == 2 ? k_lds2 : i == 3 ? k_lds3 : i == 4 ? k_lds4 : k_lds5;
  };
  auto v_at = [&](auto j) -> char* {
    constexpr int i = decltype(j)::value % NS;
    return i == 0 ? v_lds0 : i == 1 ? v_lds1 : i == 2 ? v_lds2 : i == 3 ? v_lds3 : i == 4 ? v_lds4 : v_lds5;
  };
  auto k_pick = [&](int i) -> char* {
    if (NS > 3 && i >= 3) return i == 3 ? k_lds3 : i == 4 ? k_lds4 : k_lds5;
    return i == 0 ? k_lds0 : i == 1 ? k_lds1 : k_lds2;
  };
  auto v_pick = [&](int i) -> char* {
    if (NS > 3 && i >= 3) return i == 3 ? v_lds3 : i == 4 ? v_lds4 : v_lds5;
    return i == 0 ? v_lds0 : i == 1 ? v_lds1 : v_lds2;
  };

  // Parameters that only a segment's ends need are read again there: held over
  // the tile loop they would push its scalars into vector registers.
  auto late = []() -> const RowsParams& {
    typedef const __attribute__((address_space(4))) RowsParams* Kernarg;
    Kernarg at = (Kernarg)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const RowsParams*)at;
  };

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row_part = wave % kRowParts, key_part = wave / kRowParts;
  const bool loads_k = wave < kLoaders;
  const GroupDivider by_group(p.group);
  const int page_row_bytes = p.kv_heads * kRowBytes;
  const float c2 = p.scale_log2;

  const Plan plan = plan_units<kTree, kGroupRows, kBlockThreads>(p, lists);
  const int run = run_of_workgroup();
  int unit = min(run, plan.total / plan.per_run + 1) * plan.per_run;
  const int unit_end = min(plan.total, unit + plan.per_run);

  while (unit < unit_end) {
    const Segment g = find_segment<kTree, kGroupRows>(p, lists, unit, unit_end);
    // Lane values are derived anew in every segment: kept over the loop they
    // would take registers that the tile loop needs.
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int n = lane & 31, half = lane >> 5;

    // What needs no page number is loaded first: the selection, then Q.
    const int32_t* chosen = nullptr;
    int entry = 0;
    if constexpr (!kTree) {
      chosen = selection_of(p, g);
      entry = selection_entry(p, chosen);
    }
    // ---- rows ----
    const int rows = min(kGroupRows, g.tokens * p.group - g.row_base);
    const bool active = 32 * row_part < rows;
    i16x8_t q[8];
    {
      const int row = 32 * row_part + n;
      const int token = by_group.token(g.row_base + row);
      const int head = g.row_base + row - token * p.group;
      const bool ok = row < rows;
      const uint16_t* const src = p.query + (int64_t)(g.row0 + (ok ? token : 0)) * p.query_stride +
                                  (int64_t)(g.kv_head * p.group + (ok ? head : 0)) * kHeadDim + 8 * half;
#pragma unroll
      for (int c = 0; c < 8; ++c) q[c] = *reinterpret_cast<const i16x8_t*>(src + 16 * c);
    }
    __builtin_amdgcn_sched_barrier(0);

    // ---- the steps of the segment ----
    // Step t < list_tiles is keys kStep (t % kSteps) .. of page t / kSteps of the
    // list; a tree's own steps follow.  All have kStep valid keys but the list's
    // last, which has `cut`, and the tree's last.
    int list_pages;
    bool in_lds = false;
    int list_tiles, cut, tiles_end;
    if constexpr (kTree) {
      list_pages = g.units - 1;
      list_tiles = (g.context + kStep - 1) / kStep;
      cut = g.context - (list_tiles - 1) * kStep;
      tiles_end = g.hi == g.units ? list_tiles + (g.tokens + kStep - 1) / kStep : kSteps * g.hi;
    } else {
      list_pages = selected_list<kBlockThreads>(p, lists, g, chosen, entry, in_lds);
    }
    auto logical_of = [&](int i) {  // page i of the list, i uniform
      if constexpr (kTree) return i;
      else return in_lds ? __builtin_amdgcn_readfirstlane(lists.list[i]) : __builtin_amdgcn_readlane(entry, i & 63);
    };
    if constexpr (!kTree) {
      const int end = g.pos0 + g.tokens;  // behind the block's last row
      const int held = list_pages > 0 ? min(kPageSize, end - logical_of(list_pages - 1) * kPageSize) : 0;
      list_tiles = list_pages > 0 ? kSteps * (list_pages - 1) + (held + kStep - 1) / kStep : 0;
      cut = held - (held - 1) / kStep * kStep;
      tiles_end = min(kSteps * g.hi, list_tiles);
    }
    const int t0 = kSteps * g.lo;
    const int tiles = max(0, tiles_end - t0);
    // The leading tiles that every row attends whole.
    int plain;
    if constexpr (kTree) {
      plain = min(g.context / kStep, tiles_end) - t0;
    } else {
      const int first = max(g.pos0, 0);  // the first row's position
      int pages = min(g.hi, list_pages);
      while (pages > g.lo && logical_of(pages - 1) * kPageSize + kPageSize - 1 > first) --pages;
      plain = kSteps * (pages - g.lo);
      if (pages < min(g.hi, list_pages) && pages >= g.lo) {
        plain += max(0, (first + 1 - logical_of(pages) * kPageSize) / kStep);
      }
      plain = min(plain, tiles);
    }

    // ---- page numbers: 64 pages a register, block b in the one of its parity ----
    bool bad_pages = false;  // some page of those loaded is none of the cache
    auto load_pages = [&](int block) {
      const int i = 64 * block + lane;
      int phys = -1;
      bool bad = false;
      if (i < list_pages) {
        int logical = i;
        if constexpr (!kTree) logical = in_lds ? lists.list[i] : entry;
        const RowsParams& l = late();
        phys = l.block_table[g.request * l.table_stride + logical];
        if (phys >= l.num_pages) phys = -1;
        if (phys < 0) bad = true;
      }
      bad_pages |= __any(bad) != 0;
      return phys;
    };
    const int block0 = g.lo >> 6;
    int phys_even = load_pages(block0 + (block0 & 1));
    int phys_odd = load_pages(block0 + 1 - (block0 & 1));
    auto phys_of = [&](int page) {
      return __builtin_amdgcn_readlane((page >> 6) & 1 ? phys_odd : phys_even, page & 63);
    };
    int refill_tile = kSteps * (64 * (block0 + 1) + 32);  // K of this tile on its way: the block after next is due
    auto refill = [&](int t) {
      if (__builtin_expect(t >= refill_tile, 0)) {
        const int block = t / (64 * kSteps) + 1;
        int phys = load_pages(block);
        asm volatile("" : "+v"(phys));  // landed before the paths join
        if (block & 1) phys_odd = phys; else phys_even = phys;
        refill_tile += 64 * kSteps;
      }
    };

    // ---- DMA: this wave's share of a tile of K or V ----
    const int dma_row = 4 * kDmaShare * (wave % kLoaders) + (lane >> 4);
    // Lane i of instruction j fills slot i % 16 of key row dma_row + 4 j, which
    // holds chunk k_slot or v_slot of the row.
    const int dma_chunk = 16 * (loads_k ? k_slot(dma_row, lane & 15) : v_slot(dma_row, lane & 15));
    const int dma_turn = loads_k ? 64 : 0;
    static_assert(kDmaShare <= 4, "the rows of a wave's instructions differ in bits 2 and 3");
    const char* const cache = (loads_k ? p.key_cache : p.value_cache) + g.kv_head * kRowBytes;
    const int64_t page_stride = loads_k ? p.key_page_stride : p.value_page_stride;
    const int draft_rb = kTree ? (int)(loads_k ? p.draft_key_stride : p.draft_value_stride) : 0;
    const char* const draft =
        kTree ? (loads_k ? p.draft_key : p.draft_value) + (int64_t)g.row0 * draft_rb + g.kv_head * kRowBytes : nullptr;
    // Tile t of the list or tree; past the segment's end an empty range.
    auto source = [&](int t, int& rb) {
      const char* base;
      rb = page_row_bytes;
      int valid = t == list_tiles - 1 ? cut : kStep;
      if (kTree && t >= list_tiles) {
        const int at = (t - list_tiles) * kStep;
        rb = draft_rb;
        base = draft + (int64_t)at * draft_rb;
        valid = min(g.tokens - at, kStep);
      } else {
        const int phys = phys_of(t / kSteps);
        base = cache + max(phys, 0) * page_stride + (t % kSteps) * (kStep * page_row_bytes);
        if (phys < 0) valid = 0;
      }
      if (t >= tiles_end) valid = 0;
      return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, valid > 0 ? (valid - 1) * rb + kRowBytes : 0,
                                               kBufferFlags);
    };
    auto dma = [&](__amdgpu_buffer_rsrc_t rsrc, int rb, char* slot, int j) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, TM_LDS(slot + ((wave % kLoaders) * kDmaShare + j) * 1024), 16,
                                               (unsigned)((dma_row + 4 * j) * rb + (dma_chunk ^ (dma_turn * j))), 0, 0, 0);
    };
    auto load_tile = [&](int t, char* slot) {
      int rb;
      const __amdgpu_buffer_rsrc_t rsrc = source(t, rb);
#pragma unroll
      for (int j = 0; j < kDmaShare; ++j) dma(rsrc, rb, slot, j);
    };
    if (loads_k) {
      load_tile(t0, k_lds0);
      load_tile(t0 + 1, k_lds1);
      load_tile(t0 + 2, k_lds2);
      if (NS > 3) load_tile(t0 + 3, k_lds3);
      if (NS > 4) {
        load_tile(t0 + 4, k_lds4);
        load_tile(t0 + 5, k_lds5);
      }
    } else {
      load_tile(t0, v_lds0);
      load_tile(t0 + 1, v_lds1);
      if (NS > 3) load_tile(t0 + 2, v_lds2);
      if (NS > 4) {
        load_tile(t0 + 3, v_lds3);
        load_tile(t0 + 4, v_lds4);
      }
    }

    // ---- operand addresses in a slot ----
    int k_off = key_part * kTileBytes + n * kRowBytes + 16 * k_slot(n, half);
    const int v_key = 4 * half + ((lane & 15) >> 2);
    const int v_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    int v_off = key_part * kTileBytes + v_key * kRowBytes + 16 * v_slot(v_key, v_dim >> 3) + 2 * (v_dim & 7);

    float m_run = -INFINITY, l_run = 0.0f;  // of the row; the sum over this lane's keys
    f32x16_t o[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) o[m] = f32x16_t{};
    // The row's running max takes in a tile's; returns the exponentials' shift.
    auto raise = [&](float top) {
      if (__any(top > m_run + kLazyRescale)) {
        const float m_new = fmaxf(m_run, top);
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int m = 0; m < 4; ++m) o[m] *= alpha;
        m_run = m_new;
      }
      return m_run == -INFINITY ? 0.0f : m_run;
    };
    auto row_top = [&](const f32x16_t& s) {
      float top = s[0];
#pragma unroll
      for (int v = 1; v < 16; ++v) top = fmaxf(top, s[v]);
      return half_max(top) * c2;
    };
    auto scores = [&](const char* ks) {
      f32x16_t s = f32x16_t{};
      i16x8_t kf[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) kf[c] = k_operand_of(ks, k_off, c);
#pragma unroll
      for (int c = 0; c < 8; ++c) s = Type::mfma32(kf[c], q[c], s);
      return s;
    };

    // ---- the pipeline ----
    // The first `plain` tiles; `next`: this wave's next tile to load.
    int next = loads_k ? NS : NS - 1;
    if (plain > 0) {
      if (loads_k) wait_dma_but<(NS - 1) * kDmaShare>();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      f32x16_t s_a = f32x16_t{}, s_b = f32x16_t{};
      float top = -INFINITY;
      if (active) {
        s_a = scores(k_lds0);
        if (bad_pages && phys_of(t0 / kSteps) < 0) s_a = f32x16_t{} - INFINITY;
        top = row_top(s_a);
      }
      // Iteration it, it % NS = j: scores of tile it in s_cur, their row max in
      // `top`; K of it + NS and V of it + NS - 1 go into the slots just read.
      auto iteration = [&](auto j, int it, f32x16_t& s_cur, f32x16_t& s_nxt) {
        constexpr int J = decltype(j)::value;
        const char* const kr = k_at(Index<J + 1>{});
        const char* const vr = v_at(Index<J>{});
        wait_dma_but<(NS - 2) * kDmaShare>();  // K of it + 1, V of it have landed
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();  // for every wave, and the slots that are filled next are read
        asm volatile("" ::: "memory");
        const int t_load = t0 + it + (loads_k ? NS : NS - 1);
        refill(t_load);
        int rb;
        const __amdgpu_buffer_rsrc_t src = source(t_load, rb);
        char* const slot = loads_k ? k_at(Index<J>{}) : v_at(Index<J + NS - 1>{});
        asm volatile("" : "+v"(k_off), "+v"(v_off));  // addresses are formed here, not held over the loop
        if (!active) {
#pragma unroll
          for (int j = 0; j < kDmaShare; ++j) dma(src, rb, slot, j);
          return;
        }
        const float shift = raise(top);
        i16x8_t kf[8], va[8];
        float px[16], sum = 0.0f;
        auto expo = [&](int e) {
          px[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s_cur[e], c2, -shift));
          sum += px[e];
        };
#pragma unroll
        for (int k = 0; k < kAhead; ++k) kf[k] = k_operand_of(kr, k_off, k);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k % (8 / kDmaShare) == 0) dma(src, rb, slot, k / (8 / kDmaShare));
          if (k + kAhead < 8) kf[k + kAhead] = k_operand_of(kr, k_off, k + kAhead);
          else va[k + kAhead - 8] = v_operand_of(vr, v_off, k + kAhead - 8);
          s_nxt = Type::mfma32(kf[k], q[k], k == 0 ? f32x16_t{} : s_nxt);
          expo(k);
          if ((k & 1) == 0) expo(8 + (k >> 1));
          __builtin_amdgcn_sched_barrier(0);
        }
        typename Type::vec pb[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) pb[0][e] = (elem)px[e];
        asm volatile("" ::"v"(pb[0]), "v"(px[8]), "v"(px[9]), "v"(px[10]), "v"(px[11]), "v"(sum));
        if (__builtin_expect(bad_pages, 0)) {
          if (phys_of((t0 + it + 1) / kSteps) < 0) s_nxt = f32x16_t{} - INFINITY;  // a page without keys
        }
        float next = -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k + kAhead < 8) va[k + kAhead] = v_operand_of(vr, v_off, k + kAhead);
          if (k < 4) {
            expo(12 + k);
            if (k == 3) {
#pragma unroll
              for (int e = 8; e < 16; ++e) pb[1][e - 8] = (elem)px[e];
            }
          }
          o[k & 3] = Type::mfma32(va[k], __builtin_bit_cast(i16x8_t, pb[k >> 2]), o[k & 3]);
          next = fmaxf(fmaxf(next, s_nxt[2 * k]), s_nxt[2 * k + 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
        l_run += sum;
        top = half_max(next) * c2;
      };
      const int fast = plain - 1;
      for (int it = 0; it < fast;) {
        iteration(Index<0>{}, it, s_a, s_b);
        if (++it == fast) break;
        iteration(Index<1>{}, it, s_b, s_a);
        if (++it == fast) break;
        iteration(Index<2>{}, it, s_a, s_b);
        if (++it == fast) break;
        iteration(Index<3>{}, it, s_b, s_a);
        if (++it == fast) break;
        if constexpr (kUnroll == 6) {
          iteration(Index<4>{}, it, s_a, s_b);
          if (++it == fast) break;
          iteration(Index<5>{}, it, s_b, s_a);
          ++it;
        }
      }
      next += fast;
      // The last of them: its scores are there, no tile of the pipeline follows.
      wait_dma();
      __syncthreads();
      if (active) {
        if (fast & 1) s_a = s_b;
        const char* const vr = v_pick(fast % NS);
        const float shift = raise(top);
        typename Type::vec pb[2];
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s_a[e], c2, -shift));
          sum += x;
          pb[e >> 3][e & 7] = (elem)x;
        }
        l_run += sum;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          o[k & 3] = Type::mfma32(v_operand_of(vr, v_off, k), __builtin_bit_cast(i16x8_t, pb[k >> 2]), o[k & 3]);
        }
      }
    }

    // ---- the rest, with masks, one tile after the other ----
    int tail_lane = threadIdx.x & 63;
    asm volatile("" : "+v"(tail_lane));
    const int my_row = 32 * row_part + (tail_lane & 31);
    const int my_token = by_group.token(g.row_base + my_row);
    const bool my_ok = my_row < rows;
    uint64_t my_mask = 0;
    if constexpr (kTree) {
      if (my_ok) my_mask = (uint64_t)late().tree_mask[g.row0 + my_token];
    }
    for (int it = max(plain, 0); it < tiles; ++it) {
      wait_dma();
      __syncthreads();
      const int t = t0 + it;
      const int turn = it % NS;
      // the slots of the tiles before this one are free
      for (; next < min(it + NS, tiles); ++next) load_tile(t0 + next, loads_k ? k_pick(next % NS) : v_pick(next % NS));
      if (!active) continue;
      const char* const ks = k_pick(turn);
      const char* const vs = v_pick(turn);
      f32x16_t s = scores(ks);
      // All tiles here have a mask; the condition, always true, keeps it a block of its
      // own for the scheduler (32 fp16 trees of 12-24 nodes: 82.5 us, without it 85).
      if (it >= plain) {
        int thr = -1;  // the last key offset in the tile that the row attends
        uint32_t bits = ~0u;
        if (kTree && t >= list_tiles) {
          const int at = (t - list_tiles) * kStep + key_part * kKvTile;
          thr = g.tokens - 1 - at;
          bits = (uint32_t)(my_mask >> (at & 63));
        } else if (phys_of(t / kSteps) >= 0) {
          if constexpr (kTree) {
            thr = g.context - 1 - t * kStep - key_part * kKvTile;
          } else {
            thr = (my_ok ? g.pos0 + my_token : -1) - logical_of(t / kSteps) * kPageSize - (t % kSteps) * kStep -
                  key_part * kKvTile;
          }
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int key = elem_key(v) + 4 * half;
          const bool seen = key <= thr && ((bits >> key) & 1) != 0;
          s[v] = seen ? s[v] : -INFINITY;
        }
      }
      const float shift = raise(row_top(s));
      typename Type::vec pb[2];
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c2, -shift));
        sum += x;
        pb[e >> 3][e & 7] = (elem)x;
      }
      l_run += sum;
      i16x8_t va[8];
      typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));
      u16x8_t size = {};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        va[k] = v_operand_of(vs, v_off, k);
        size = __builtin_elementwise_max(size, __builtin_bit_cast(u16x8_t, va[k] & (short)0x7fff));
      }
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) bad |= size[e] >= Type::kExp;
      if (__builtin_expect(!__any(bad), 1)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k & 3] = Type::mfma32(va[k], __builtin_bit_cast(i16x8_t, pb[k >> 2]), o[k & 3]);
      } else {
        // The finite entries, then for each other kind the product of indicators
        // (such an entry; the key attended, whatever its weight rounded to).
        i16x8_t attended[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) attended[e >> 3][e & 7] = s[e] != -INFINITY ? Type::kOne : 0;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
          for (int kind = 0; kind < 4; ++kind) {  // finite, +inf, -inf, NaN
            f32x16_t has = f32x16_t{};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // read anew and opaque: kept over the kinds they would spill
              asm volatile("" ::: "memory");
              u32x4_t a = __builtin_bit_cast(u32x4_t, v_operand_of(vs, v_off, m + 4 * j));
              asm volatile("" : "+v"(a));
#pragma unroll
              for (int e = 0; e < 4; ++e) a[e] = only_kind<Type>(a[e], kind) | only_kind<Type>(a[e] >> 16, kind) << 16;
              if (kind == 0) o[m] = Type::mfma32(__builtin_bit_cast(i16x8_t, a), __builtin_bit_cast(i16x8_t, pb[j]), o[m]);
              else has = Type::mfma32(__builtin_bit_cast(i16x8_t, a), attended[j], has);
            }
            if (kind > 0) {
              // opaque: the compiler takes no operand for a NaN; +inf and -inf give one by themselves
              float odd = __uint_as_float(kind == 1 ? 0x7f800000u : kind == 2 ? 0xff800000u : 0x7fc00000u);
              asm volatile("" : "+v"(odd));
#pragma unroll
              for (int v = 0; v < 16; ++v) o[m][v] += has[v] > 0.0f ? odd : 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
    m_run = row_shift(m_run, half_sum(l_run));
    wait_dma();
    __syncthreads();  // no slot is read or written any more

    // ---- the key parts' sums: the second's through LDS ----
    if constexpr (KP == 2) {
      char* const at = row_part < NS ? k_pick(row_part) : v_pick(row_part - NS);
      float* const sums = reinterpret_cast<float*>(v_pick(NS - 1)) + 2 * (64 * row_part + lane);
      static_assert(kRowParts - NS < NS - 1 && 64 * 64 * 4 <= kStepBytes, "a wave's O fits a slot");
      if (active && key_part == 1) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x4_t x = {o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2],
                             o[i >> 2][4 * (i & 3) + 3]};
          *reinterpret_cast<f32x4_t*>(at + (64 * i + lane) * 16) = x;
        }
        sums[0] = m_run;
        sums[1] = l_run;
      }
      __syncthreads();
      if (active && key_part == 0) {
        const float other = sums[0];
        const float top = fmaxf(m_run, other);
        const float shift = top == -INFINITY ? 0.0f : top;
        const float w0 = __builtin_amdgcn_exp2f(m_run - shift), w1 = __builtin_amdgcn_exp2f(other - shift);
        l_run = l_run * w0 + sums[1] * w1;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x4_t x = *reinterpret_cast<const f32x4_t*>(at + (64 * i + lane) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i >> 2][4 * (i & 3) + e] = o[i >> 2][4 * (i & 3) + e] * w0 + x[e] * w1;
        }
        m_run = top;
      }
    }
    const bool writes = active && key_part == 0;

    // Rows out: normalised and rounded, gathered in the wave's slot as whole
    // rows (8-byte pieces in, 16-byte chunks out, chunk c of row r at c ^ (r %
    // 16)), stored through L2 in whole cache lines.
    char* const stage = wave < NS ? k_pick(wave) : v_pick(wave - NS);
    auto store_rows = [&](float l) {
      const RowsParams& q = late();
      const float l_row = half_sum(l);
      const float inv = l_row > 0.0f ? 1.0f / l_row : 0.0f;
      typedef elem elem4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int m = 0; m < 4; ++m) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          elem4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = (elem)(o[m][4 * c + e] * inv);
          *reinterpret_cast<elem4*>(stage + n * kRowBytes + 16 * ((4 * m + c) ^ (n & 15)) + 8 * half) = y;
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 4 * j + (lane >> 4), c = lane & 15;
        const u32x4_t y = *reinterpret_cast<const u32x4_t*>(stage + r * kRowBytes + 16 * (c ^ (r & 15)));
        const int row = 32 * row_part + r;
        const int t = by_group.token(g.row_base + row);
        const int h = g.row_base + row - t * q.group;
        if (row < rows && t >= g.held) {
          *reinterpret_cast<u32x4_t*>(q.out + ((int64_t)(g.row0 + t) * q.heads + g.kv_head * q.group + h) * kHeadDim +
                                      8 * c) = y;
        }
      }
    };
    if (g.lo == 0 && g.hi == g.units) {
      if (writes) store_rows(l_run);
    } else {
      // ---- a group of several runs ----
      const Shared shared(g, plan.per_run);
      const __amdgpu_buffer_rsrc_t rec = __builtin_amdgcn_make_buffer_rsrc(
          (void*)late().partials, (short)0, (int)((unsigned)late().workgroups * 2u * kRecordBytes), kBufferFlags);
      // record: O [wave][d-block, quarter][lane][4], then row maxima and lane sums [wave][lane]
      auto piece = [&](int i) { return (unsigned)(((row_part * 16 + i) * 64 + lane) * 16); };
      const unsigned at_max = (unsigned)(kGroupRows * kHeadDim * 4 + (row_part * 64 + lane) * 4);
      const unsigned at_sum = at_max + kRowParts * 64 * 4;
      if (writes) {
        const unsigned own = shared.record(run, kRecordBytes);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x4_t x = {o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2],
                             o[i >> 2][4 * (i & 3) + 3]};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), rec, own + piece(i), 0, kCpolAgent);
        }
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(m_run), rec, own + at_max, 0, kCpolAgent);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l_run), rec, own + at_sum, 0, kCpolAgent);
      }
      if (last_to_arrive(late(), shared, &s_last) && writes) {
        float top = -INFINITY, l = 0.0f;
#pragma unroll
        for (int m = 0; m < 4; ++m) o[m] = f32x16_t{};
        // two partials' loads in flight at a time
        for (int r = shared.first_run; r <= shared.last_run; r += 2) {
          float mr[2], lr[2];
          f32x4_t x[2][16];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // past the last one its loads fall outside the buffer's range
            const unsigned from =
                r + j <= shared.last_run ? shared.record(r + j, kRecordBytes) : kOutOfRange;
            mr[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rec, from + at_max, 0, kCpolAgent));
            lr[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rec, from + at_sum, 0, kCpolAgent));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              x[j][i] = __builtin_bit_cast(f32x4_t,
                                           __builtin_amdgcn_raw_buffer_load_b128(rec, from + piece(i), 0, kCpolAgent));
            }
          }
          if (r + 1 > shared.last_run) mr[1] = -INFINITY;
          const float next = fmaxf(top, fmaxf(mr[0], mr[1]));
          const float shift = next == -INFINITY ? 0.0f : next;
          const float keep = __builtin_amdgcn_exp2f(top - shift);
          const float w0 = __builtin_amdgcn_exp2f(mr[0] - shift), w1 = __builtin_amdgcn_exp2f(mr[1] - shift);
          l = l * keep + lr[0] * w0 + lr[1] * w1;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[i >> 2][4 * (i & 3) + e] = o[i >> 2][4 * (i & 3) + e] * keep + x[0][i][e] * w0 + x[1][i][e] * w1;
            }
          }
          top = next;
        }
        store_rows(l);
      }
    }
    unit = g.first + g.hi;
    __syncthreads();
  }
}

template <class Type, bool kTree>
hipError_t launch_type(const RowsParams& p, int shape_rows, hipStream_t stream) {
  const dim3 grid((unsigned)p.workgroups);
  if (shape_rows == kBlockRows) {
    hipLaunchKernelGGL((blocks_attention_kernel<Type, 8, 1, kTree>), grid, dim3(512), 0, stream, p);
  } else if (kTree || p.workgroups <= kComputeUnits) {
    hipLaunchKernelGGL((blocks_attention_kernel<Type, 8, 2, kTree>), grid, dim3(512), 0, stream, p);
  } else if constexpr (!kTree) {
    hipLaunchKernelGGL((blocks_attention_kernel<Type, 4, 1, kTree>), grid, dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_blocks_attention(const RowsParams& p, int shape_rows, bool fp16, hipStream_t stream) {
  if (p.selected == nullptr) {
    return fp16 ? launch_type<Fp16, true>(p, shape_rows, stream) : launch_type<Bf16, true>(p, shape_rows, stream);
  }
  return fp16 ? launch_type<Fp16, false>(p, shape_rows, stream) : launch_type<Bf16, false>(p, shape_rows, stream);
}

}  // namespace tmx
