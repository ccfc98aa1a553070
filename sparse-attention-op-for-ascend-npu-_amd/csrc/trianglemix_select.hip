// Key bounds of KV pages, and the selection of pages by them, for MI355X
// (gfx950).
//
// Bounds: the elementwise smallest and largest key of each page and KV head, in
// the keys' own type, so nothing is rounded.  The pages that hold a request's
// last tokens are reduced again from the cache as a whole, so the result does
// not depend on what they held before.
//
// Selection: for a block of up to 32 query rows and a KV head,
//   score(page) = max over the heads h of the group of
//                 sum_d (qs_hd >= 0 ? qs_hd * max_d : qs_hd * min_d),
// qs_h the sum of the block's rows: no key of the page has a larger dot product
// with qs_h.  Scores are summed in 64 bits: the 16-bit inputs leave nothing
// (or next to nothing) to round there, so which page comes last of those
// chosen does not hang on the order of a sum.  A score is kept as a 64-bit
// integer key of the same order: 0 no candidate, 1 a score that is not a
// number (ranks last), all ones a page that is always taken.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_pages.h"

namespace tmx {
namespace {

typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// 16-bit floats as signed integers of the same order.  NaNs lie above +inf and
// below -inf.
__device__ __forceinline__ s16x8_t ordered(s16x8_t x) { return x ^ ((x >> 15) & (short)0x7fff); }

constexpr int kBoundsThreads = 256;
constexpr int kRowsAtOnce = kBoundsThreads / 16;  // 16 lanes read one token's 256 bytes

// One workgroup per (request, one of its last pages, KV head): 32 KB of keys,
// all of a thread's loads in flight at once.
template <bool kFp16>
__global__ void __launch_bounds__(kBoundsThreads) page_bounds_kernel(const BoundsParams p) {
  const int kv_head = blockIdx.y, b = blockIdx.z;
  const int seq = min(max(p.seq_lens[b], 0), p.table_cols * kPageSize);
  const int first = max(0, seq - p.num_tokens);
  const int page = first / kPageSize + (int)blockIdx.x;
  const int held = min(kPageSize, seq - page * kPageSize);
  if (held <= 0) return;
  const int phys = p.block_table[b * p.table_stride + page];
  if (phys < 0 || phys >= p.num_pages) return;
  const int sub = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const uint16_t* const keys = p.key_cache + phys * p.page_stride + (int64_t)kv_head * kHeadDim + 8 * sub;
  const int64_t stride = (int64_t)p.kv_heads * kHeadDim;
  s16x8_t x[kPageSize / kRowsAtOnce];
#pragma unroll
  for (int i = 0; i < kPageSize / kRowsAtOnce; ++i) {
    // rows past the last token repeat it: they change neither bound
    x[i] = *reinterpret_cast<const s16x8_t*>(keys + min(r0 + kRowsAtOnce * i, held - 1) * stride);
  }
  s16x8_t lo = ordered(x[0]), hi = lo;
#pragma unroll
  for (int i = 1; i < kPageSize / kRowsAtOnce; ++i) {
    const s16x8_t y = ordered(x[i]);
    lo = __builtin_elementwise_min(lo, y);
    hi = __builtin_elementwise_max(hi, y);
  }
  __shared__ s16x8_t s_lo[kRowsAtOnce][16], s_hi[kRowsAtOnce][16];
  s_lo[r0][sub] = lo;
  s_hi[r0][sub] = hi;
  __syncthreads();
  if (threadIdx.x < 16) {
#pragma unroll
    for (int i = 1; i < kRowsAtOnce; ++i) {
      lo = __builtin_elementwise_min(lo, s_lo[i][sub]);
      hi = __builtin_elementwise_max(hi, s_hi[i][sub]);
    }
    constexpr short kInf = kFp16 ? 0x7c00 : 0x7f80;
    constexpr short kNan = kFp16 ? 0x7e00 : 0x7fc0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // a NaN among the keys makes both bounds NaN (-inf is ~kInf in this order)
      if (hi[e] > kInf || lo[e] < (short)~kInf) lo[e] = hi[e] = kNan;
    }
    const int64_t at = ((int64_t)phys * p.kv_heads + kv_head) * kHeadDim + 8 * sub;
    *reinterpret_cast<s16x8_t*>(p.page_min + at) = ordered(lo);
    *reinterpret_cast<s16x8_t*>(p.page_max + at) = ordered(hi);
  }
}

template <bool kFp16>
__device__ __forceinline__ float to_float(short x) {
  return kFp16 ? (float)__builtin_bit_cast(_Float16, x) : __uint_as_float((unsigned)(uint16_t)x << 16);
}

// The sums of each block's rows, one thread per (block, head, dim).
constexpr int kPoolThreads = 256;
template <bool kFp16>
__global__ void __launch_bounds__(kPoolThreads) pool_rows_kernel(const SelectParams p) {
  const int64_t i = (int64_t)blockIdx.x * kPoolThreads + threadIdx.x;
  const int width = p.heads * kHeadDim;
  const int64_t block = i / width;
  if (block >= (int64_t)p.requests * p.slab_blocks) return;
  const int b = p.request0 + (int)(block / p.slab_blocks);
  const int t0 = (p.block0 + (int)(block % p.slab_blocks)) * kSelectRows;
  const int pos0 = max(p.seq_lens[b], 0) - p.rows;
  const uint16_t* src = p.query + (int64_t)b * p.rows * p.query_stride + i % width;
  double sum = 0.0;
  for (int t = max(t0, -pos0); t < min(t0 + kSelectRows, p.rows); ++t) {
    sum += (double)to_float<kFp16>((short)src[t * p.query_stride]);
  }
  p.pooled[i] = sum;
}

// Adds the 16 lanes of a row, the result in all of them.
template <int kCtrl>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, 0xf, 0xf, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), kCtrl, 0xf, 0xf, true);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double sum16(double x) {
  x = dpp_add<0xb1>(x);   // quad_perm 1 0 3 2
  x = dpp_add<0x4e>(x);   // quad_perm 2 3 0 1
  x = dpp_add<0x141>(x);  // row_half_mirror
  return dpp_add<0x140>(x);  // row_mirror
}

__device__ __forceinline__ uint64_t score_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  if ((u & 0x7fffffffffffffffull) > 0x7ff0000000000000ull) return 1;
  return (int64_t)u < 0 ? ~u : u | 0x8000000000000000ull;
}

// 16 lanes hold one page's bounds (8 dims each), PP pages in turn, and run
// over the blocks and heads.
constexpr int kScoreThreads = 256;
template <bool kFp16, int PP>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const SelectParams p) {
  const int sub = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const int kv_head = blockIdx.y % p.kv_heads, slab_b = blockIdx.y / p.kv_heads;
  const int b = p.request0 + slab_b;
  const int page0 = ((int)blockIdx.x * (kScoreThreads / 16) + slot) * PP;
  const int group = p.heads / p.kv_heads;
  const int seq = max(p.seq_lens[b], 0);
  const int pages = min(p.table_cols, (seq + kPageSize - 1) / kPageSize);
  if ((int)blockIdx.x * (kScoreThreads / 16) * PP >= pages) return;
  float lo[PP][8], hi[PP][8];
  bool there[PP];
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    const int phys = page0 + i < pages ? p.block_table[b * p.table_stride + page0 + i] : -1;
    there[i] = phys >= 0 && phys < p.num_pages;
    const int64_t at = ((int64_t)(there[i] ? phys : 0) * p.kv_heads + kv_head) * kHeadDim + 8 * sub;
    const s16x8_t l = *reinterpret_cast<const s16x8_t*>(p.page_min + at);
    const s16x8_t h = *reinterpret_cast<const s16x8_t*>(p.page_max + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[i][e] = to_float<kFp16>(l[e]);
      hi[i][e] = to_float<kFp16>(h[e]);
    }
  }
  for (int blk = blockIdx.z; blk < p.slab_blocks; blk += gridDim.z) {
    uint64_t best[PP];
#pragma unroll
    for (int i = 0; i < PP; ++i) best[i] = 0;
    for (int g = 0; g < group; ++g) {
      const int head = kv_head * group + g;
      double q[8];
      if (p.pooled) {
        const double* src = p.pooled + (((int64_t)slab_b * p.slab_blocks + blk) * p.heads + head) * kHeadDim + 8 * sub;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = src[e];
      } else {
        const s16x8_t x =
            *reinterpret_cast<const s16x8_t*>(p.query + b * p.query_stride + (int64_t)head * kHeadDim + 8 * sub);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = (double)to_float<kFp16>(x[e]);
      }
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fma(q[e], (double)(q[e] >= 0.0 ? hi[i][e] : lo[i][e]), sum);
        const uint64_t key = score_key(sum16(sum));
        best[i] = key > best[i] ? key : best[i];
      }
    }
    if (sub == 0) {
      uint64_t* const dst =
          p.scores + (((int64_t)slab_b * p.slab_blocks + blk) * p.kv_heads + kv_head) * p.table_cols;
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        if (page0 + i < pages) dst[page0 + i] = there[i] ? best[i] : 0;
      }
    }
  }
}

// The `count` largest keys of one (block, KV head), the lowest page first among
// equal ones, written in the order of the pages.  A key's threshold is found by
// halving: as soon as exactly `count` keys lie at or above the middle it is
// done (about 14 steps for 1024 pages); only equal keys take it down to one
// value.
constexpr int kTopThreads = 256;
template <int KPT>
__global__ void __launch_bounds__(kTopThreads) top_pages_kernel(const SelectParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x;  // of the slab: (request * blocks + block) * kv_heads + head
  const int kv_head = row % p.kv_heads;
  const int blk = p.block0 + row / p.kv_heads % p.slab_blocks;
  const int b = p.request0 + row / p.kv_heads / p.slab_blocks;
  const int pos0 = max(p.seq_lens[b], 0) - p.rows;
  const int last = pos0 + min(p.rows, (blk + 1) * kSelectRows) - 1;
  const int first = max(0, pos0 + blk * kSelectRows);
  const int pages = last < 0 ? 0 : min(p.table_cols, last / kPageSize + 1);
  const int recent = first / kPageSize - p.recent_pages + 1;
  const uint64_t* const src = p.scores + (int64_t)row * p.table_cols;
  int32_t* const out = p.out + (((int64_t)b * p.blocks + blk) * p.kv_heads + kv_head) * p.count;
  __shared__ int s_sum[2][kTopThreads / 64];
  int turn = 0;
  auto total = [&](int mine) {  // of one count per wave, the same in every lane
    if (lane == 0) s_sum[turn][wave] = mine;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kTopThreads / 64; ++w) sum += s_sum[turn][w];
    turn ^= 1;
    return sum;
  };
  // key i of a thread is page i * 256 + threadIdx.x
  uint64_t key[KPT];
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int page = i * kTopThreads + threadIdx.x;
    key[i] = page < pages ? src[page] : 0;
    if (key[i] != 0 && p.recent_pages > 0 && page >= recent) key[i] = ~0ull;
    if (key[i] != 0 && page < p.sink_pages) key[i] = ~0ull;
  }
  auto at_least = [&](uint64_t bound) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < KPT; ++i) n += __popcll(__ballot(key[i] >= bound));
    return total(n);
  };
  uint64_t bound = 1;  // keys at or above it are taken
  uint64_t equal = 0;  // and of the keys equal to this, the first `rest`
  int rest = 0;
  if (at_least(1) > p.count) {
    uint64_t low = 1, high = ~0ull;  // more than count keys >= low, at most count >= high
    int above = at_least(high);
    while (above < p.count && high - low > 1) {
      const uint64_t mid = low + (high - low) / 2;
      const int n = at_least(mid);
      if (n > p.count) {
        low = mid;
      } else {
        high = mid;
        above = n;
      }
    }
    bound = high;
    if (above < p.count) {
      equal = low;
      rest = p.count - above;
    }
  }
  int written = 0, ties = 0;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    if (i * kTopThreads >= pages) break;
    bool take = key[i] >= bound;
    if (rest > 0) {
      const bool tie = key[i] == equal;
      const uint64_t mask = __ballot(tie);
      __syncthreads();
      if (lane == 0) s_sum[0][wave] = __popcll(mask);
      __syncthreads();
      int before = ties + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
      for (int w = 0; w < kTopThreads / 64; ++w) {
        before += w < wave ? s_sum[0][w] : 0;
        ties += s_sum[0][w];
      }
      take |= tie && before < rest;
    }
    const uint64_t mask = __ballot(take);
    __syncthreads();
    if (lane == 0) s_sum[0][wave] = __popcll(mask);
    __syncthreads();
    int at = written + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
    for (int w = 0; w < kTopThreads / 64; ++w) {
      at += w < wave ? s_sum[0][w] : 0;
      written += s_sum[0][w];
    }
    if (take) out[at] = i * kTopThreads + threadIdx.x;
  }
  for (int i = written + threadIdx.x; i < p.count; i += kTopThreads) out[i] = -1;
}

template <bool kFp16>
hipError_t launch_select(const SelectParams& p, hipStream_t stream) {
  const int64_t row_blocks = (int64_t)p.requests * p.slab_blocks;
  if (p.pooled) {
    const int64_t n = row_blocks * p.heads * kHeadDim;
    hipLaunchKernelGGL(pool_rows_kernel<kFp16>, dim3((unsigned)((n + kPoolThreads - 1) / kPoolThreads)),
                       dim3(kPoolThreads), 0, stream, p);
  }
  constexpr int kSlots = kScoreThreads / 16;
  if (p.slab_blocks > 1) {
    const unsigned chunks = (unsigned)((p.table_cols + 4 * kSlots - 1) / (4 * kSlots));
    const unsigned split = (unsigned)min(p.slab_blocks, 8);
    hipLaunchKernelGGL((score_kernel<kFp16, 4>), dim3(chunks, (unsigned)(p.requests * p.kv_heads), split),
                       dim3(kScoreThreads), 0, stream, p);
  } else {
    const unsigned chunks = (unsigned)((p.table_cols + kSlots - 1) / kSlots);
    hipLaunchKernelGGL((score_kernel<kFp16, 1>), dim3(chunks, (unsigned)(p.requests * p.kv_heads), 1),
                       dim3(kScoreThreads), 0, stream, p);
  }
  const dim3 grid((unsigned)(row_blocks * p.kv_heads));
  if (p.table_cols <= 4 * kTopThreads) {
    hipLaunchKernelGGL(top_pages_kernel<4>, grid, dim3(kTopThreads), 0, stream, p);
  } else if (p.table_cols <= 16 * kTopThreads) {
    hipLaunchKernelGGL(top_pages_kernel<16>, grid, dim3(kTopThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL(top_pages_kernel<64>, grid, dim3(kTopThreads), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_page_bounds(const BoundsParams& p, bool fp16, hipStream_t stream) {
  const int64_t most = ((int64_t)p.num_tokens - 1 + kPageSize - 1) / kPageSize + 1;
  const dim3 grid((unsigned)(most < p.table_cols ? most : p.table_cols), (unsigned)p.kv_heads, (unsigned)p.batch);
  if (fp16) {
    hipLaunchKernelGGL(page_bounds_kernel<true>, grid, dim3(kBoundsThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL(page_bounds_kernel<false>, grid, dim3(kBoundsThreads), 0, stream, p);
  }
  return hipGetLastError();
}

hipError_t launch_select_pages(const SelectParams& p, bool fp16, hipStream_t stream) {
  return fp16 ? launch_select<true>(p, stream) : launch_select<false>(p, stream);
}

}  // namespace tmx
