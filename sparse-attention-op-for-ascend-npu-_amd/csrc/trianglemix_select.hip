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

// The sums of each block's rows: four threads per (block, head, 8 dims), each
// with eight rows' loads in flight, joined through LDS.
constexpr int kPoolThreads = 256;
constexpr int kPoolColumns = 64;
template <bool kFp16>
__global__ void __launch_bounds__(kPoolThreads) pool_rows_kernel(const SelectParams p) {
  __shared__ double s_sum[3][8][kPoolColumns];
  const int quarter = threadIdx.x / kPoolColumns, column = threadIdx.x % kPoolColumns;
  const int64_t i = (int64_t)blockIdx.x * kPoolColumns + column;
  const int width = p.heads * (kHeadDim / 8);
  const int block = (int)(i / width);
  const bool real = block < p.requests * p.slab_blocks;
  const int at = (int)(i % width) * 8;
  double sum[8] = {};
  if (real) {
    const int b = p.request0 + block / p.slab_blocks;
    const int t0 = (p.block0 + block % p.slab_blocks) * kSelectRows + 8 * quarter;
    const uint16_t* const src = p.query + (int64_t)b * p.rows * p.query_stride + at;
    const int seq = p.seq_lens[b];
    s16x8_t x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const s16x8_t*>(src + min(t0 + j, p.rows - 1) * p.query_stride);
    const int begin = p.rows - max(seq, 0);  // the first row of the request
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool row = t0 + j >= begin && t0 + j < p.rows;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += row ? (double)to_float<kFp16>(x[j][e]) : 0.0;
    }
  }
  if (quarter > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s_sum[quarter - 1][e][column] = sum[e];
  }
  __syncthreads();
  if (quarter > 0 || !real) return;
  double* const dst = p.pooled + (int64_t)block * p.heads * kHeadDim + at;
#pragma unroll
  for (int e = 0; e < 8; ++e) dst[e] = (sum[e] + s_sum[0][e][column]) + (s_sum[1][e][column] + s_sum[2][e][column]);
}

__device__ __forceinline__ uint64_t score_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  if ((u & 0x7fffffffffffffffull) > 0x7ff0000000000000ull) return 1;
  return (int64_t)u < 0 ? ~u : u | 0x8000000000000000ull;
}

// max(x, 0) and min(x, 0) of finite numbers by the sign bit.
__device__ __forceinline__ double positive(double x) { return __builtin_signbit(x) ? 0.0 : x; }
__device__ __forceinline__ double negative(double x) { return __builtin_signbit(x) ? x : 0.0; }
__device__ __forceinline__ bool odd_number(double x) {
  return (__builtin_bit_cast(uint64_t, x) & 0x7ff0000000000000ull) == 0x7ff0000000000000ull;
}
__device__ __forceinline__ void keep_larger(uint64_t& x, uint64_t y) { x = y > x ? y : x; }

// The scores as 64-bit matrix products, q+ max + q- min with q+ = max(q, 0), q-
// = min(q, 0): lane l of a wave holds the bounds of page l % 16 of 16, of every
// 32 dims the eight from 8 (l / 16) on, and the products run over tiles of
// rows, block * padded + head with the group padded to a power of two.
// Infinities and NaNs, which a product with zero would turn into NaN, take a
// plain loop: the rows that hold one for all pages, the pages that hold one by
// themselves, so that a page's score does not hang on its neighbours' bounds (the two
// forms may differ in the last bit).
typedef double f64x4_t __attribute__((ext_vector_type(4)));
typedef double f64x2_t __attribute__((ext_vector_type(2)));
constexpr int kScoreWaves = 4;
constexpr int kScoreThreads = kScoreWaves * 64;

struct Bounds16 {  // a lane's 32 dims of its page
  s16x8_t lo[4], hi[4];
};
__device__ __forceinline__ Bounds16 load_bounds(const SelectParams& p, int64_t at) {
  Bounds16 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.lo[i] = *reinterpret_cast<const s16x8_t*>(p.page_min + at + 32 * i);
    x.hi[i] = *reinterpret_cast<const s16x8_t*>(p.page_max + at + 32 * i);
  }
  return x;
}
// Bit j: some bound of the wave's page j is no finite number.
template <bool kFp16>
__device__ __forceinline__ unsigned odd_bounds(const Bounds16& x) {
  typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));
  u16x8_t most = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x8_t, x.lo[i] & (short)0x7fff));
    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x8_t, x.hi[i] & (short)0x7fff));
  }
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) odd |= most[e] >= (kFp16 ? 0x7c00 : 0x7f80);
  uint64_t lanes = __ballot(odd);
  lanes |= lanes >> 32;
  lanes |= lanes >> 16;
  return (unsigned)lanes & 0xffffu;
}
// The plain sum over a row of 128 (plus and minus its parts, from 8 quad on), in
// all four lanes of a page.  The bounds come anew from memory: nothing is kept in
// registers for this path.
template <bool kFp16>
__device__ double plain_score(const SelectParams& p, int64_t at, const double* plus, const double* minus) {
  double y = 0.0;
#pragma unroll 1
  for (int i = 0; i < 32; ++i) {
    const int d = 32 * (i >> 3) + (i & 7);
    const double q = plus[d] + minus[d];
    const uint16_t bound = q >= 0.0 ? p.page_max[at + d] : p.page_min[at + d];
    y = __builtin_fma(q, (double)to_float<kFp16>((short)bound), y);
  }
  y += __shfl_xor(y, 16);
  y += __shfl_xor(y, 32);
  return y;
}

// Up to four rows (a decoding step: one block, up to four heads a group):
// v_mfma_f64_4x4x4, its four blocks taking four pages each.  A wave runs over
// `tiles` tiles of 16 pages, one tile's bounds ahead; what bounds it is reading
// them and their conversion to 64 bits.
template <bool kFp16>
__global__ void __launch_bounds__(kScoreThreads, 4) score_few_kernel(const SelectParams p, int padded_bits, int tiles) {
  __shared__ __attribute__((aligned(16))) double s_plus[4][kHeadDim + 2], s_minus[4][kHeadDim + 2];
  __shared__ int s_odd[kScoreWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int padded = 1 << padded_bits;
  const int col = lane & 15, quad = lane >> 4;
  const int kv_head = blockIdx.x, slab_b = blockIdx.y;
  const int b = p.request0 + slab_b;
  const int group = p.heads / p.kv_heads;
  const int page0 = ((int)blockIdx.z * kScoreWaves + wave) * 16 * tiles;
  // the wave's pages, one a lane; the length is not waited for
  int phys = page0 + lane < p.table_cols && lane < 16 * tiles ? p.block_table[b * p.table_stride + page0 + lane] : -1;
  if (phys >= p.num_pages) phys = -1;
  const int seq = min(max(p.seq_lens[b], 0), p.table_cols * kPageSize);
  {
    // one row a wave, two dims a lane
    const int blk = wave >> padded_bits, g = wave & (padded - 1), head = kv_head * group + g;
    f64x2_t x = {0.0, 0.0};
    if (blk < p.slab_blocks && g < group) {
      if (p.pooled) {
        x = *reinterpret_cast<const f64x2_t*>(
            p.pooled + ((int64_t)(slab_b * p.slab_blocks + blk) * p.heads + head) * kHeadDim + 2 * lane);
      } else {
        const unsigned two =
            *reinterpret_cast<const unsigned*>(p.query + b * p.query_stride + (int64_t)head * kHeadDim + 2 * lane);
        x = f64x2_t{(double)to_float<kFp16>((short)two), (double)to_float<kFp16>((short)(two >> 16))};
      }
    }
    *reinterpret_cast<f64x2_t*>(&s_plus[wave][2 * lane]) = f64x2_t{positive(x[0]), positive(x[1])};
    *reinterpret_cast<f64x2_t*>(&s_minus[wave][2 * lane]) = f64x2_t{negative(x[0]), negative(x[1])};
    const bool odd = __any(odd_number(x[0]) || odd_number(x[1]));
    if (lane == 0) s_odd[wave] = odd ? 1 : 0;
  }
  // The lane's page in tile t, -1 for none.  Another lane holds it, so every lane
  // must be active here: one that is masked off gives a zero, page 0.
  auto page_of = [&](int t) { return __shfl(phys, 16 * t + col); };
  auto place = [&](int page) {  // an unused page's bounds are those of page 0
    return ((int64_t)max(page, 0) * p.kv_heads + kv_head) * kHeadDim + 8 * quad;
  };
  int next_page = page_of(0);
  Bounds16 next = load_bounds(p, place(next_page));
  __syncthreads();
  const bool odd_rows = (s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3]) != 0;
  const int pages = (seq + kPageSize - 1) / kPageSize;
  for (int t = 0; t < tiles; ++t) {
    if (page0 + 16 * t >= pages) return;
    Bounds16 x = next;
    const int here = next_page;
    const int64_t at = place(here);
    if (t + 1 < tiles) {
      next_page = page_of(t + 1);
      next = load_bounds(p, place(next_page));
    }
    double sum = 0.0;
    const unsigned plain = odd_rows ? 0xffffu : odd_bounds<kFp16>(x);  // pages that take the plain loop
    if (__builtin_expect(!odd_rows, 1)) {
      double c[4] = {};
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const int d = 8 * quad + 32 * (i >> 3) + (i & 7);
        const f64x2_t plus = *reinterpret_cast<const f64x2_t*>(&s_plus[lane & 3][d]);
        const f64x2_t minus = *reinterpret_cast<const f64x2_t*>(&s_minus[lane & 3][d]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const double hi = (double)to_float<kFp16>(x.hi[i >> 3][(i & 7) + j]);
          const double lo = (double)to_float<kFp16>(x.lo[i >> 3][(i & 7) + j]);
          c[2 * j] = __builtin_amdgcn_mfma_f64_4x4x4f64(plus[j], hi, c[2 * j], 0, 0, 0);
          c[2 * j + 1] = __builtin_amdgcn_mfma_f64_4x4x4f64(minus[j], lo, c[2 * j + 1], 0, 0, 0);
        }
      }
      sum = (c[0] + c[1]) + (c[2] + c[3]);
    }
    if (__builtin_expect(plain != 0, 0)) {
      for (int r = 0; r < 4; ++r) {
        const double y = plain_score<kFp16>(p, at, &s_plus[r][8 * quad], &s_minus[r][8 * quad]);
        sum = r == quad && (plain >> col & 1) != 0 ? y : sum;
      }
    }
    // row `quad` of page `col`: max over the heads of a block
    uint64_t best = (quad & (padded - 1)) < group ? score_key(sum) : 0;
    if (padded >= 2) keep_larger(best, __shfl_xor(best, 16));
    if (padded >= 4) keep_larger(best, __shfl_xor(best, 32));
    const int page = page0 + 16 * t + col;
    if ((quad & (padded - 1)) == 0 && quad < p.slab_blocks * padded && page < pages) {
      p.scores[((int64_t)(slab_b * p.slab_blocks + (quad >> padded_bits)) * p.kv_heads + kv_head) * p.table_cols + page] =
          here >= 0 ? best : 0;
    }
  }
}

// Many rows: tiles of 16 rows, v_mfma_f64_16x16x4, two tiles' query sums in LDS,
// q+ and q- apart: the loop over the products has no other instructions, which
// would not run beside 64-bit MFMAs.  A wave keeps the bounds of its 16 pages,
// converted, over all its row tiles.
template <bool kFp16>
__global__ void __launch_bounds__(kScoreThreads, 2) score_kernel(const SelectParams p, int padded_bits, int split_bits) {
  // rows of 128 and two doubles, so that 16 rows' reads meet different banks
  __shared__ __attribute__((aligned(16))) double s_plus[2][16][kHeadDim + 2], s_minus[2][16][kHeadDim + 2];
  __shared__ int s_odd[2];  // some value of the tile is no finite number
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int padded = 1 << padded_bits;
  const int col = lane & 15, quad = lane >> 4;
  const int kv_head = (int)blockIdx.x >> split_bits, slab_b = blockIdx.y;
  const int b = p.request0 + slab_b;
  const int group = p.heads / p.kv_heads;
  const int page = ((int)blockIdx.z * kScoreWaves + wave) * 16 + col;
  const int phys = page < p.table_cols ? p.block_table[b * p.table_stride + page] : -1;
  const int seq = min(max(p.seq_lens[b], 0), p.table_cols * kPageSize);

  const int rows = p.slab_blocks * padded;
  const int tile_bits = max(0, padded_bits - 4), tiles_per_block = 1 << tile_bits;
  const int row_tiles = (rows + 15) / 16;
  // Two dims a thread of four of the tile's rows; zeros for rows of the padding.
  auto fetch = [&](int row0, f64x2_t* x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + wave + 4 * j;
      const int blk = row >> padded_bits, g = row & (padded - 1);
      x[j] = f64x2_t{0.0, 0.0};
      if (row < rows && g < group) {
        const int head = kv_head * group + g;
        if (p.pooled) {
          x[j] = *reinterpret_cast<const f64x2_t*>(
              p.pooled + ((int64_t)(slab_b * p.slab_blocks + blk) * p.heads + head) * kHeadDim + 2 * lane);
        } else {
          const unsigned two =
              *reinterpret_cast<const unsigned*>(p.query + b * p.query_stride + (int64_t)head * kHeadDim + 2 * lane);
          x[j] = f64x2_t{(double)to_float<kFp16>((short)two), (double)to_float<kFp16>((short)(two >> 16))};
        }
      }
    }
  };
  auto put = [&](int buffer, const f64x2_t* x) {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      odd |= odd_number(x[j][0]) || odd_number(x[j][1]);
      *reinterpret_cast<f64x2_t*>(&s_plus[buffer][wave + 4 * j][2 * lane]) = f64x2_t{positive(x[j][0]), positive(x[j][1])};
      *reinterpret_cast<f64x2_t*>(&s_minus[buffer][wave + 4 * j][2 * lane]) = f64x2_t{negative(x[j][0]), negative(x[j][1])};
    }
    if (odd) s_odd[buffer] = 1;
  };
  // A workgroup's row tiles: whole blocks, dealt over the splits.
  const int stride = tiles_per_block << split_bits;
  int t = ((int)blockIdx.x & ((1 << split_bits) - 1)) * tiles_per_block;
  f64x2_t x[4];
  fetch(t * 16, x);
  const bool there = phys >= 0 && phys < p.num_pages;
  const int64_t at = ((int64_t)(there ? phys : 0) * p.kv_heads + kv_head) * kHeadDim + 8 * quad;
  const Bounds16 raw = load_bounds(p, at);
  if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  __syncthreads();
  put(0, x);
  const int pages = (seq + kPageSize - 1) / kPageSize;
  if ((int)blockIdx.z * kScoreWaves * 16 >= pages) return;
  const unsigned odd_pages = odd_bounds<kFp16>(raw);
  double lo[32], hi[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    lo[i] = (double)to_float<kFp16>(raw.lo[i >> 3][i & 7]);
    hi[i] = (double)to_float<kFp16>(raw.hi[i >> 3][i & 7]);
  }

  uint64_t best[4] = {0, 0, 0, 0};
  for (int buffer = 0; t < row_tiles; buffer ^= 1) {
    __syncthreads();  // the tile is in its buffer, the other buffer is read
    const int next = ((t + 1) & (tiles_per_block - 1)) == 0 ? t + 1 - tiles_per_block + stride : t + 1;
    const bool more = next < row_tiles;
    if (more) fetch(next * 16, x);
    const int row0 = t * 16;
    f64x4_t sum = {0.0, 0.0, 0.0, 0.0};
    const unsigned plain = __builtin_amdgcn_readfirstlane(s_odd[buffer]) != 0 ? 0xffffu : odd_pages;
    if (__builtin_expect(plain != 0xffffu, 1)) {
      // Physical row r of the operand is row 4 (r % 4) + r / 4 of the tile, so
      // that a lane's four results are rows 4 quad .. 4 quad + 3.
      const double* const plus = &s_plus[buffer][4 * (col & 3) + (col >> 2)][8 * quad];
      const double* const minus = &s_minus[buffer][4 * (col & 3) + (col >> 2)][8 * quad];
      f64x4_t c0 = sum, c1 = sum;
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const f64x2_t x = *reinterpret_cast<const f64x2_t*>(plus + 32 * (i >> 3) + (i & 7));
        const f64x2_t y = *reinterpret_cast<const f64x2_t*>(minus + 32 * (i >> 3) + (i & 7));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          c0 = __builtin_amdgcn_mfma_f64_16x16x4f64(x[j], hi[i + j], c0, 0, 0, 0);
          c1 = __builtin_amdgcn_mfma_f64_16x16x4f64(y[j], lo[i + j], c1, 0, 0, 0);
        }
      }
      sum = c0 + c1;
    }
    if (__builtin_expect(plain != 0, 0)) {
      for (int r = 0; r < 16; ++r) {
        const double y = plain_score<kFp16>(p, at, &s_plus[buffer][r][8 * quad], &s_minus[buffer][r][8 * quad]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = r == 4 * quad + i && (plain >> col & 1) != 0 ? y : sum[i];
      }
    }
    // max over the heads of a block: rows of a lane, then of lanes, then of tiles
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (((row0 + 4 * quad + i) & (padded - 1)) < group) keep_larger(best[i], score_key(sum[i]));
    }
    if (((t + 1) & (tiles_per_block - 1)) == 0) {
      int step = 1;  // rows that one key of a lane stands for
      if (padded >= 2) {
        keep_larger(best[0], best[1]);
        keep_larger(best[2], best[3]);
        step = 2;
      }
      if (padded >= 4) {
        keep_larger(best[0], best[2]);
        step = 4;
      }
      if (padded >= 8) keep_larger(best[0], __shfl_xor(best[0], 16));
      if (padded >= 16) keep_larger(best[0], __shfl_xor(best[0], 32));
      const int block_row0 = ((t >> tile_bits) << tile_bits) * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = block_row0 + 4 * quad + i;
        if (i % step == 0 && (row & (padded - 1)) == 0 && row < rows && page < pages) {
          p.scores[((int64_t)(slab_b * p.slab_blocks + (row >> padded_bits)) * p.kv_heads + kv_head) * p.table_cols + page] =
              there ? best[i] : 0;
        }
        best[i] = 0;
      }
    }
    if (more) {
      if (threadIdx.x == 0) s_odd[buffer ^ 1] = 0;
      __syncthreads();
      put(buffer ^ 1, x);
    }
    t = next;
  }
}

// The `count` largest keys of one (block, KV head), the lowest page first among
// equal ones, written in the order of the pages.  The threshold is found by
// counting keys in 256 bins between the smallest and the largest key, then in
// the bin that holds it: two levels or three for 1024 pages, eight at most.
constexpr int kTopThreads = 256;
static_assert(64 * kTopThreads >= kMaxTableCols, "a workgroup holds a row's keys");
// Largest value of the wave's lanes, in all of them.
template <int kCtrl>
__device__ __forceinline__ unsigned dpp_max(unsigned x) {
  const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, 0xf, 0xf, true);
  return y > x ? y : x;
}
__device__ __forceinline__ unsigned wave_max(unsigned x) {
  x = dpp_max<0xb1>(x);   // quad_perm 1 0 3 2
  x = dpp_max<0x4e>(x);   // quad_perm 2 3 0 1
  x = dpp_max<0x141>(x);  // row_half_mirror
  x = dpp_max<0x140>(x);  // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = a[0] > a[1] ? a[0] : a[1];
  const auto c = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return c[0] > c[1] ? c[0] : c[1];
}

template <int KPT>
__global__ void __launch_bounds__(kTopThreads) top_pages_kernel(const SelectParams p) {
  constexpr int W = kTopThreads / 64;
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
  __shared__ int s_sum[2][W];
  __shared__ unsigned s_key[2][W];
  __shared__ unsigned s_bins[2][256];
  int turn = 0;
  // One count per wave to their sum, and the sum of the waves before.
  auto total = [&](int mine, int* before) {
    if (lane == 0) s_sum[turn][wave] = mine;
    __syncthreads();
    int sum = 0, ahead = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      ahead += w < wave ? s_sum[turn][w] : 0;
      sum += s_sum[turn][w];
    }
    turn ^= 1;
    if (before) *before = ahead;
    return sum;
  };
  // key i of a thread is page 256 i + threadIdx.x
  uint64_t key[KPT];
  unsigned most = 0, most_neg = 0;  // largest high word, and complement, of the keys that are not always taken
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int page = i * kTopThreads + (int)threadIdx.x;
    key[i] = page < pages ? src[page] : 0;
  }
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const int page = i * kTopThreads + (int)threadIdx.x;
    if (key[i] != 0) {
      if ((p.recent_pages > 0 && page >= recent) || page < p.sink_pages) {
        key[i] = ~0ull;
      } else {
        const unsigned word = (unsigned)(key[i] >> 32);
        most = word > most ? word : most;
        most_neg = ~word > most_neg ? ~word : most_neg;
      }
    }
  }
  most = wave_max(most);
  most_neg = wave_max(most_neg);
  if (lane == 0) {
    s_key[0][wave] = most;
    s_key[1][wave] = most_neg;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) {
    most = s_key[0][w] > most ? s_key[0][w] : most;
    most_neg = s_key[1][w] > most_neg ? s_key[1][w] : most_neg;
  }
  uint64_t bound = 1;  // keys at or above it are taken
  uint64_t equal = 0;  // and of the keys equal to this, the first `rest`
  int rest = 0;
  int candidates = 0, above = 0;  // keys, and those always taken
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    candidates += __popcll(__ballot(key[i] != 0));
    above += __popcll(__ballot(key[i] == ~0ull));
  }
  candidates = total(candidates, nullptr);
  above = total(above, nullptr);
  if (candidates > p.count) {
    // The keys in [low, high) hold the last one taken.  A level counts them in
    // 256 bins and goes on in the bin in which the count is reached.
    uint64_t low = (uint64_t)~most_neg << 32 | (most_neg == ~0u ? 1 : 0), high = ((uint64_t)most + 1) << 32;
    for (int level = 0; above < p.count; level ^= 1) {
      const int shift = max(0, 56 - __clzll((long long)(high - low - 1)));
      s_bins[level][threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        if (key[i] >= low && key[i] < high) atomicAdd(&s_bins[level][(key[i] - low) >> shift], 1);
      }
      __syncthreads();
      // bins 4 lane .. 4 lane + 3, and how many keys lie in them and the bins above
      int bin[4], upto = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bin[j] = s_bins[level][4 * lane + j];
        upto += bin[j];
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int add = __shfl_down(upto, d);
        if (lane + d < 64) upto += add;
      }
      // the last lane whose bins and those above reach the count, and in it the bin
      const int at_lane = 63 - __clzll((long long)__ballot(above + upto >= p.count));
      int j_at = 0, reached = above + upto, over = reached;
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        over -= bin[j];  // keys above bin j
        if (over >= p.count) {
          j_at = j + 1;
          reached = over;
        }
      }
      const int j = __builtin_amdgcn_readlane(j_at, at_lane);
      const int with = __builtin_amdgcn_readlane(reached, at_lane);
      const int in_bin = __builtin_amdgcn_readlane(j_at == 0 ? bin[0] : j_at == 1 ? bin[1] : j_at == 2 ? bin[2] : bin[3], at_lane);
      low += (uint64_t)(4 * at_lane + j) << shift;
      if (with == p.count) {
        bound = low;
        above = with;
      } else {
        above = with - in_bin;
        if (shift == 0) {
          bound = low + 1;
          equal = low;
          rest = p.count - above;
          break;
        }
        high = low + (1ull << shift);
      }
    }
    if (bound == 1) bound = high;  // all that are taken always are
  }
  auto below = [](uint64_t mask) {  // set bits under this lane
    return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
  };
  int written = 0, ties = 0;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    if (i * kTopThreads >= pages) break;
    bool take = key[i] >= bound;
    int before;
    if (rest > 0) {
      const bool tie = key[i] == equal;
      const uint64_t mask = __ballot(tie);
      const int all = total(__popcll(mask), &before);
      take |= tie && ties + before + below(mask) < rest;
      ties += all;
    }
    const uint64_t mask = __ballot(take);
    const int all = total(__popcll(mask), &before);
    // a workspace that others write to meanwhile may show more keys always taken than fit
    const int at = written + before + below(mask);
    if (take && at < p.count) out[at] = i * kTopThreads + (int)threadIdx.x;
    written += all;
  }
  for (int i = written + threadIdx.x; i < p.count; i += kTopThreads) out[i] = -1;
}

template <bool kFp16>
hipError_t launch_select(const SelectParams& p, hipStream_t stream) {
  const int64_t row_blocks = (int64_t)p.requests * p.slab_blocks;
  if (p.pooled) {
    const int64_t n = row_blocks * p.heads * (kHeadDim / 8);
    hipLaunchKernelGGL(pool_rows_kernel<kFp16>, dim3((unsigned)((n + kPoolColumns - 1) / kPoolColumns)),
                       dim3(kPoolThreads), 0, stream, p);
  }
  int padded_bits = 0;
  while ((1 << padded_bits) < p.heads / p.kv_heads) ++padded_bits;
  const int padded = 1 << padded_bits;
  const int rows = p.slab_blocks * padded;
  const unsigned requests = (unsigned)p.requests, kv_heads = (unsigned)p.kv_heads;
  if (rows <= 4) {
    // Two tiles of pages a wave once that still gives every SIMD four waves.
    // Chunks of pages last: workgroups go round the 8 XCDs, and the chunks past
    // a request's length have no work.
    const unsigned wide = (unsigned)((p.table_cols + 32 * kScoreWaves - 1) / (32 * kScoreWaves));
    const int tiles = wide * kv_heads * requests >= 1024 ? 2 : 1;
    const unsigned chunks = (unsigned)((p.table_cols + 16 * tiles * kScoreWaves - 1) / (16 * tiles * kScoreWaves));
    hipLaunchKernelGGL(score_few_kernel<kFp16>, dim3(kv_heads, requests, chunks), dim3(kScoreThreads), 0, stream, p,
                       padded_bits, tiles);
  } else {
    // Row tiles are dealt over enough workgroups for two waves per SIMD: the
    // bounds of a wave's pages are converted once per wave.
    const unsigned chunks = (unsigned)((p.table_cols + 16 * kScoreWaves - 1) / (16 * kScoreWaves));
    const int units = (rows + (padded > 16 ? padded : 16) - 1) / (padded > 16 ? padded : 16);
    int split_bits = 0;
    while ((2 << split_bits) <= units && (chunks * kv_heads * requests << split_bits) < 512) ++split_bits;
    hipLaunchKernelGGL(score_kernel<kFp16>, dim3(kv_heads << split_bits, requests, chunks), dim3(kScoreThreads), 0,
                       stream, p, padded_bits, split_bits);
  }
  const unsigned n = (unsigned)(row_blocks * p.kv_heads);
  if (p.table_cols <= kTopThreads) {
    hipLaunchKernelGGL(top_pages_kernel<1>, dim3(n), dim3(kTopThreads), 0, stream, p);
  } else if (p.table_cols <= 4 * kTopThreads) {
    hipLaunchKernelGGL(top_pages_kernel<4>, dim3(n), dim3(kTopThreads), 0, stream, p);
  } else if (p.table_cols <= 16 * kTopThreads) {
    hipLaunchKernelGGL(top_pages_kernel<16>, dim3(n), dim3(kTopThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL(top_pages_kernel<64>, dim3(n), dim3(kTopThreads), 0, stream, p);
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
