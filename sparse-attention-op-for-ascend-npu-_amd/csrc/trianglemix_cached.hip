// Attention of the last tokens of each request over its paged cache, of e4m3
// numbers or of the queries' own 16-bit type, for MI355X (gfx950).
//
// Work.  The rows are those of a request's last tokens, few enough for the waves of
// a workgroup (trianglemix_chunks.hip has the others): all heads of a GQA group times
// the tokens, numbered token * G + head.  A workgroup is four or eight waves, each
// with a tile of 16 NT rows: of neighbouring KV heads (their numbers lie side by side
// in memory, 128 bytes of e4m3 each: read by one workgroup they stream at 5.9 TB/s,
// by one each at 4.6 to 5.7), of several row tiles, or with parts of the keys.  A group
// is what a workgroup so covers.  Its 32-key tiles are the first `sinks` keys' and
// those from the window's first key on, or all; others are not read.
//
// Shares.  Every group's tiles are cut into equal shares, as many as the GPU holds
// workgroups over all groups: lengths are read on the device, the grid does not
// depend on them, a workgroup has one share.  (Equal runs over all groups in a row
// keep the workgroups more even, but each then ends two or three groups, and pays
// for the join of the waves, the partial and the next start each time: 64
// requests of 2000 to 16384 tokens 222 us, with runs 225 to 240; a window of 512
// keys 27 and 40.)  Partials are merged as in trianglemix_cached_device.h.
//
// K and V go from memory into registers, a tile ahead of the one in use: a wave loads
// what it multiplies itself, so the loop has neither LDS nor barriers.  More tiles
// ahead (two, three), two workgroups a CU and waves held together by a barrier a tile
// were no faster: 64 to 128 KB in flight a CU are enough.  The waves' sums meet in LDS behind the loop.
//
// What bounds it: memory.  64 requests of 2000 to 16384 tokens (1.22 GB) 220 us, four
// of 65536 to 131072 (0.83 GB) 148, at 5.6 TB/s over all and 5.9 within the loop; the
// rest is the start (lengths, table and first tiles, each waiting for the one before: 3
// us), the join and the merge (5 to 10).  One token of 8111 on two KV heads: 10.3
// us, launch and round trips alone.
//
// Contractions (per wave, 32 keys x 16 NT rows, v_mfma_f32_16x16x32)
//   S^T (keys x rows) = K Q^T     A = K, B = Q
//   O^T (dims x rows) += V^T P^T  A = V^T, B = P
// Lane l holds row l % 16.  The keys of S^T's two 16-key halves u are dealt so that
// accumulator element i of half u in lanes of quad l / 16 is key 8 quad + 4 u + i:
// the lane's eight scores are its eight k-slots of P.  V^T wants, for one dim, eight
// keys in a lane: lane l loads dims 8 (l % 16) .. + 7 of keys 8 quad .. + 7, a
// block of 8 x 8 that it transposes in registers (v_perm); product m has the dims
// 8 i + m (i the operand's row), so that a lane's results are 32 dims in a row.
// e4m3 numbers become 16-bit ones on the way (v_cvt_scalef32_pk, exact): K of the
// queries' type, V fp16 with fp16 weights.
//
// Numerics: scores, row max, row sum and O in fp32, exponentials as exp2 of
// scores in units of log2(e); the weights are rounded for the PV product alone.
// fp16 weights are 2^7 times themselves (at most 2^15, as the row max may be stale
// by 2^8): what is 2^-31 of the largest is still a number, so that millions of
// small ones are not lost.  Keys past a page's valid ones are not read (the
// buffer's range ends there and gives zeros).  In tiles where some row masks a key,
// V entries that are not finite are kept out of the product and added only to rows
// that attend them.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_cached_device.h"

namespace tmx {
namespace {

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

// Sum over the wave, and over its lanes up to this one: lanes 1, 2, 4 and 8 back in
// their row of 16, then a row's last lane to the rows behind it (a move each in
// place of a round trip through LDS: with divide_up 0.5 us a call less).
template <int kControl, int kRowMask>
__device__ __forceinline__ int moved(int x) {
  return __builtin_amdgcn_update_dpp(0, x, kControl, kRowMask, 0xf, false);
}
__device__ __forceinline__ int wave_prefix(int x) {
  x += moved<0x111, 0xf>(x);  // row_shr:1
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);  // row_bcast:15
  x += moved<0x143, 0xc>(x);  // row_bcast:31
  return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_prefix(x), 63); }

// a / b rounded up, for a + b below 2^21: the quotient of a + b - 1/2 in 32 bits is off by less
// than it is from the next whole number.
__device__ __forceinline__ int divide_up(int a, int b) {
  return (int)(((float)(a + b) - 0.5f) * __builtin_amdgcn_rcpf((float)b));
}

// A wave's share of a page, 32 keys: what its lanes load, and the operands made of it.
template <class Type, CacheType kCache>
struct Tile;

template <class Type>
struct Tile<Type, CacheType::kSame> {
  typedef Type Weight;  // of P and V^T
  static constexpr int kElemBytes = 2;
  u32x4_t k[2][4], v[8];

  // The first of the eight dims of Q's (and K's) operand c.
  static __device__ __forceinline__ int q_dim(int c, int quad) { return 32 * c + 8 * quad; }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, const int* k_off,
                                       const int* v_off) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) k[u][c] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off[u] + 64 * c, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_off[j], 0, 0);
  }
  __device__ __forceinline__ i16x8_t k_operand(int u, int c) const { return __builtin_bit_cast(i16x8_t, k[u][c]); }
  // Dims 2 w and 2 w + 1 of key j's eight.
  __device__ __forceinline__ unsigned v_pair(int j, int w) const { return v[j][w]; }
  // Of number i in memory: 0 finite, 1 +infinity, 2 -infinity, 3 NaN.
  static __device__ __forceinline__ int odd_kind(const char* at, int i) {
    const unsigned x = reinterpret_cast<const uint16_t*>(at)[i], size = x & 0x7fffu;
    return size < Type::kExp ? 0 : size > Type::kExp ? 3 : x == size ? 1 : 2;
  }
  // Whether some V entry is no finite number.
  __device__ __forceinline__ bool odd_value() const {
    typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));
    u16x8_t size = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) size = __builtin_elementwise_max(size, __builtin_bit_cast(u16x8_t, v[j] & 0x7fff7fffu));
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) odd |= size[e] >= Type::kExp;
    return odd;
  }
  // V with zeros in the place of what is no finite number.
  __device__ __forceinline__ void keep_finite() {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const unsigned x = v[j][w];
        v[j][w] = ((x & 0x7fffu) < Type::kExp ? x & 0xffffu : 0) | ((x & 0x7fff0000u) < (Type::kExp << 16) ? x & 0xffff0000u : 0);
      }
    }
  }
};

template <class Type>
struct Tile<Type, CacheType::kE4m3> {
  typedef Fp16 Weight;
  static constexpr int kElemBytes = 1;
  u32x4_t k[2][2];
  u32x2_t v[8];

  // A 16-byte load holds two operands' dims.
  static __device__ __forceinline__ int q_dim(int c, int quad) { return 64 * (c >> 1) + 16 * quad + 8 * (c & 1); }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, const int* k_off,
                                       const int* v_off) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int c = 0; c < 2; ++c) k[u][c] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off[u] + 64 * c, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __builtin_amdgcn_raw_buffer_load_b64(vr, v_off[j], 0, 0);
  }
  __device__ __forceinline__ i16x8_t k_operand(int u, int c) const {
    const unsigned lo = k[u][c >> 1][2 * (c & 1)], hi = k[u][c >> 1][2 * (c & 1) + 1];
    const u32x4_t x = {from_e4m3<Type, false>(lo), from_e4m3<Type, true>(lo), from_e4m3<Type, false>(hi),
                       from_e4m3<Type, true>(hi)};
    return __builtin_bit_cast(i16x8_t, x);
  }
  __device__ __forceinline__ unsigned v_pair(int j, int w) const {
    return w & 1 ? from_e4m3<Fp16, true>(v[j][w >> 1]) : from_e4m3<Fp16, false>(v[j][w >> 1]);
  }
  static __device__ __forceinline__ int odd_kind(const char* at, int i) {
    return (reinterpret_cast<const uint8_t*>(at)[i] & 0x7f) == 0x7f ? 3 : 0;
  }
  __device__ __forceinline__ bool odd_value() const {
    unsigned odd = 0;  // NaN is 0x7f or 0xff: the only sizes that a one carries into the sign's place
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int w = 0; w < 2; ++w) odd |= (v[j][w] & 0x7f7f7f7fu) + 0x01010101u;
    }
    return (odd & 0x80808080u) != 0;
  }
  __device__ __forceinline__ void keep_finite() {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const unsigned odd = ((v[j][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        v[j][w] &= ~((odd >> 7) * 0xffu);
      }
    }
  }
};

// V^T of dims 8 i + 2 w and 8 i + 2 w + 1: the two operands, eight keys each.
template <class T>
__device__ __forceinline__ void v_operands(const T& tile, int w, u32x4_t& even, u32x4_t& odd) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned a = tile.v_pair(2 * j, w), b = tile.v_pair(2 * j + 1, w);
    even[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    odd[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  }
}


template <class Type, CacheType kCache, int NT, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, 1) cached_attention_kernel(const CachedParams p) {
  constexpr int kThreads = 64 * kWaves, kWaveShift = kWaves == 8 ? 3 : 2;
  typedef Tile<Type, kCache> Share;
  typedef typename Share::Weight Weight;
  typedef typename Type::elem elem;
  constexpr int kRows = 16 * NT;
  constexpr int kDepth = 2;  // tiles in registers, the one in use among them
  constexpr int kHeadBytes = kHeadDim * Share::kElemBytes;
  constexpr float kWeightBits = std::is_same_v<Weight, Fp16> ? 7.0f : 0.0f;

  __shared__ __attribute__((aligned(16))) float o_lds[kWaves][16 * kHeadDim];
  __shared__ float s_max[kWaves][kRows], s_sum[kWaves][kRows];
  __shared__ float join[kThreads][10];
  __shared__ unsigned s_odd[kWaves * kRows][3][4];  // note_odd: a bit a dim, for +infinity, -infinity, NaN
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 15;  // row of the wave's 16-row tile
  const int quad = lane >> 4;
  const int G = p.group;
  const GroupDivider by_group(p.group);
  const int token_bytes = p.kv_heads * kHeadBytes;
  // this wave's head, row tile and keys among the workgroup's
  const int slots = kWaves >> p.key_shift, slot = wave & (slots - 1), key_part = wave >> (kWaveShift - p.key_shift);
  const int row_tiles = 1 << p.row_shift, row_tile = slot & (row_tiles - 1);
  const int head_shift = kWaveShift - p.key_shift - p.row_shift, head_part = slot >> p.row_shift;
  const int head_groups = p.kv_heads >> head_shift;
  const int slot_rows = row_tiles > 1 ? kRows : min(kRows, p.rows * G);  // of a partial's record
  const int record_rows = slots * slot_rows;
  constexpr int kFlight = 8, kEach = NT;  // of the merge
  const int cluster = kFlight * merge_parts<kThreads>(record_rows);  // shares that are merged at once
  for (int i = tid; i < kWaves * kRows * 12; i += kThreads) (&s_odd[0][0][0])[i] = 0;
  __syncthreads();

  // ---- this workgroup's group, and its tiles lo .. hi - 1, one of `shares` shares ----
  // Every group is cut into as many shares as its tiles take at `least` a share, the
  // same for all and enough to keep all groups' shares within the grid.
  auto len_of = [&](int b) TM_INLINED { return b < p.batch ? max(p.seq_lens[b], 0) : 0; };
  auto tiles_of = [&](int n) TM_INLINED { return Tiles<kKvTile>(p, n - p.rows, n - 1).count; };
  int len64 = len_of(lane);
  int tiles64 = tiles_of(len64);  // of requests base .. base + 63, one a lane
  int total = tiles64;
  for (int b = 64 + lane; b < p.batch + lane; b += 64) total += tiles_of(len_of(b));
  total = wave_sum(total);
  // Sure: sum(ceil(tiles / least)) is at most total / least and a share more a group.
  // One block of requests: the smallest such number by halves from total / workgroups on.
  // (From the most tiles of a request on, every group is one share.)
  int least = max(p.min_tiles, (int)(((unsigned)(total * head_groups) + (unsigned)p.full_shares - 1u) / (unsigned)p.full_shares));
  least = min(least, kMaxTableCols * (kPageSize / kKvTile));
  if (p.batch <= 64 && least > p.min_tiles) {
    int low = max(p.min_tiles, (int)((unsigned)(total * head_groups) / (unsigned)p.workgroups));
#pragma unroll 1
    for (int i = 0; i < p.halvings && low < least; ++i) {
      const int mid = (int)(((unsigned)low + (unsigned)least) >> 1);
      const int all = wave_sum(divide_up(tiles64, mid)) * head_groups;
      if (all <= p.workgroups) least = mid;
      else low = mid + 1;
    }
  }
  const int run = blockIdx.x;
  int base = 0, before = 0, shares64, upto64;
  for (;;) {
    // no more shares than are merged at once, where that leaves them short
    const int each64 = max(least, min(divide_up(tiles64, cluster), 8 << p.key_shift));
    shares64 = divide_up(tiles64, each64);
    upto64 = before + wave_prefix(shares64 * head_groups);
    if (__builtin_amdgcn_readlane(upto64, 63) > run) break;
    before = __builtin_amdgcn_readlane(upto64, 63);
    base += 64;
    if (base >= p.batch) return;  // more workgroups than shares
    len64 = len_of(base + lane);
    tiles64 = tiles_of(len64);
  }
  const int in_block = __ffsll((unsigned long long)__ballot(upto64 > run)) - 1;
  const int request = base + in_block;
  const int len = __builtin_amdgcn_readlane(len64, in_block);
  int shares = __builtin_amdgcn_readlane(shares64, in_block);
  const int at = run - (__builtin_amdgcn_readlane(upto64, in_block) - shares * head_groups);
  // the shares of neighbouring heads side by side: they read neighbouring numbers
  const int share = __builtin_amdgcn_readfirstlane(divide_up(at + 1, head_groups)) - 1, head_group = at - share * head_groups;
  const int part_rows = p.rows * G;
  const int pos0 = len - p.rows;  // of the first token; a negative one is no row
  const Tiles<kKvTile> tiles(p, pos0, len - 1);
  const int each = __builtin_amdgcn_readfirstlane(divide_up(tiles.count, shares));  // as even as they come
  shares = __builtin_amdgcn_readfirstlane(divide_up(tiles.count, each));
  if (share >= shares) return;
  const int lo = share * each, hi = min(lo + each, tiles.count);
  const Shares group(p, p.workgroups, record_rows, run - at + head_group, head_groups, share, shares);
  const int tokens = min(len, p.table_cols * kPageSize);  // with a key
  const bool whole = shares == 1;
  const int kv_head = (head_group << head_shift) + head_part;
  const int row_base = row_tile * kRows;  // this wave's rows in the part
  const int valid_rows = min(kRows, part_rows - row_base);  // none: the wave only takes part in the joins
  const int first_pos = pos0 + by_group.token(row_base);
  const int last_pos = valid_rows > 0 ? pos0 + by_group.token(row_base + valid_rows - 1) : -1;
  const int row0 = request * p.rows;  // of query and out

  // ---- Q ----
  i16x8_t q[NT][4];
  int row_pos[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row_base + 16 * n + col;
    const int t = by_group.token(r);
    const bool ok = 16 * n + col < valid_rows;
    row_pos[n] = ok ? pos0 + t : -1;
    const uint16_t* const from =
        p.query + (int64_t)(row0 + t) * p.query_stride + (int64_t)(kv_head * G + (r - t * G)) * kHeadDim;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      q[n][c] = i16x8_t{};
      if (ok) q[n][c] = *reinterpret_cast<const i16x8_t*>(from + Share::q_dim(c, quad));
    }
  }

  float c2 = p.scale_log2;
  if constexpr (kCache == CacheType::kE4m3) c2 *= p.key_scale[kv_head];

  // ---- tiles: step i of key part k is tile lo + (i << key_shift) + k of the list ----
  const ConstInts table = (ConstInts)(p.block_table + (int64_t)request * p.table_stride);
  const int steps = ((hi - lo - 1) >> p.key_shift) + 1;
  auto tile_of = [&](int step) TM_INLINED { return tiles.tile(lo + (step << p.key_shift) + key_part); };
  auto entry = [&](int step) TM_INLINED {  // page of the cache, or -1
    int phys = -1;
    const int t = tile_of(step);
    if (lo + (step << p.key_shift) + key_part < hi && t < tiles.end) phys = table[t / (kPageSize / kKvTile)];
    return (unsigned)phys < (unsigned)p.num_pages ? phys : -1;
  };
  auto first_key = [&](int step) TM_INLINED { return tile_of(step) * kKvTile; };
  // the first key that the last row's window holds, and that the first row's does
  const int last_low = p.window < 0 ? 0 : max(last_pos, 0) - p.window;
  const int first_low = p.window < 0 ? 0 : max(first_pos, 0) - p.window;
  // Keys of the tile that are in memory, 0 where no row attends any of them.
  auto valid_keys = [&](int step, int phys) TM_INLINED {
    const int key0 = first_key(step);
    if (phys < 0 || key0 > last_pos || (key0 + 31 < first_low && key0 >= p.sinks)) return 0;
    return min(32, tokens - key0);
  };
  auto value_tile = [&](int step, int phys) TM_INLINED {
    return p.value_cache + max(phys, 0) * p.value_page_stride + kv_head * kHeadBytes + (first_key(step) % kPageSize) * token_bytes;
  };
  int k_off[2], v_off[8];
#pragma unroll
  for (int u = 0; u < 2; ++u) k_off[u] = (8 * (col >> 2) + 4 * u + (col & 3)) * token_bytes + 16 * quad;
#pragma unroll
  for (int j = 0; j < 8; ++j) v_off[j] = (8 * quad + j) * token_bytes + 8 * Share::kElemBytes * col;
  auto load = [&](Share& t, int step, int phys) TM_INLINED {
    const int valid = valid_keys(step, phys);
    const int range = valid > 0 ? (valid - 1) * token_bytes + kHeadBytes : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(p.key_cache + max(phys, 0) * p.key_page_stride + kv_head * kHeadBytes +
                (first_key(step) % kPageSize) * token_bytes),
        (short)0, range, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vr =
        __builtin_amdgcn_make_buffer_rsrc((void*)value_tile(step, phys), (short)0, range, kBufferFlags);
    t.load(kr, vr, k_off, v_off);
  };

  float m_run[NT], l_run[NT];
  f32x4_t o[8][NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m_run[n] = -INFINITY;
    l_run[n] = 0.0f;
#pragma unroll
    for (int m = 0; m < 8; ++m) o[m][n] = f32x4_t{};
  }

  // Notes the V entries of a tile that are no finite numbers for the rows that attend
  // them, apart from the product: 0 * NaN would reach the others too.
  auto note_odd = [&](int step, int phys) TM_INLINED {
    const int key0 = first_key(step), keys = valid_keys(step, phys);
    const int pos = pos0 + by_group.token(row_base + lane);  // of row `lane`
    const char* at = value_tile(step, phys);
#pragma unroll 1
    for (int k = 0; k < keys; ++k, at += token_bytes) {
      const int lower = Share::odd_kind(at, lane), upper = Share::odd_kind(at, lane + 64);
      const int key = key0 + k;
      const bool seen =
          lane < valid_rows && key <= pos && (p.window < 0 || key >= max(pos, 0) - p.window || key < p.sinks);
#pragma unroll 1
      for (int kind = 1; kind < 4; ++kind) {
        const unsigned long long lo64 = __ballot(lower == kind), hi64 = __ballot(upper == kind);
        if (seen && (lo64 | hi64) != 0) {
          unsigned* const to = s_odd[slot * kRows + lane][kind - 1];
          atomicOr(to, (unsigned)lo64);
          atomicOr(to + 1, (unsigned)(lo64 >> 32));
          atomicOr(to + 2, (unsigned)hi64);
          atomicOr(to + 3, (unsigned)(hi64 >> 32));
        }
      }
    }
  };

  auto compute = [&](Share& t, int step, int phys) TM_INLINED {
    if (valid_keys(step, phys) == 0) return;
    const int key0 = first_key(step);
    const bool masked = key0 + 31 > first_pos || (key0 < last_low && key0 + 31 >= p.sinks);
    f32x4_t s[2][NT];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[u][n] = f32x4_t{};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const i16x8_t a = t.k_operand(u, c);
#pragma unroll
        for (int n = 0; n < NT; ++n) s[u][n] = Type::mfma16(a, q[n][c], s[u][n]);
      }
    }
    if (masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int low = p.window < 0 ? 0 : max(row_pos[n], 0) - p.window;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + 8 * quad + e;
          const bool seen = key <= row_pos[n] && (key >= low || key < p.sinks);
          s[e >> 2][n][e & 3] = seen ? s[e >> 2][n][e & 3] : -INFINITY;
        }
      }
    }
    i16x8_t pb[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, s[e >> 2][n][e & 3]);
      top = row_max(top) * c2;
      if (__any(top > m_run[n] + kLazyRescale)) {
        const float m_new = fmaxf(m_run[n], top);
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run[n] - m_new);
        l_run[n] *= alpha;
#pragma unroll
        for (int m = 0; m < 8; ++m) o[m][n] *= alpha;
        m_run[n] = m_new;
      }
      const float shift = kWeightBits - (m_run[n] == -INFINITY ? 0.0f : m_run[n]);
      typename Weight::vec weight;
      float add = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][n][e & 3], c2, shift));
        add += x;
        weight[e] = (typename Weight::elem)x;
      }
      l_run[n] += add;
      pb[n] = __builtin_bit_cast(i16x8_t, weight);
    }
    if (masked && __builtin_expect(__any(t.odd_value()) != 0, 0)) {
      note_odd(step, phys);
      t.keep_finite();
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      __builtin_amdgcn_sched_barrier(0);
      u32x4_t even, odd;
      v_operands(t, w, even, odd);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[2 * w][n] = Weight::mfma16(__builtin_bit_cast(i16x8_t, even), pb[n], o[2 * w][n]);
        o[2 * w + 1][n] = Weight::mfma16(__builtin_bit_cast(i16x8_t, odd), pb[n], o[2 * w + 1][n]);
      }
    }
  };

  // Tile slot s holds step i + s; the step kDepth - 1 ahead is on its way.
  Share tile[kDepth];
  int phys[kDepth];
#pragma unroll
  for (int s = 0; s < kDepth; ++s) phys[s] = entry(s);
#pragma unroll
  for (int s = 0; s + 1 < kDepth; ++s) load(tile[s], s, phys[s]);
  for (int i = 0; i < steps; i += kDepth) {
#pragma unroll
    for (int s = 0; s < kDepth; ++s) {
      constexpr int kAhead = kDepth - 1;
      const int ahead = (s + kAhead) % kDepth;
      load(tile[ahead], i + s + kAhead, phys[ahead]);
      const int own = phys[s];
      phys[s] = entry(i + s + kDepth);
      if (i + s < steps) compute(tile[s], i + s, own);
    }
  }

  // ---- the key parts' sums, 16 rows of every slot at a time through LDS ----
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float l = row_sum(l_run[n]);
    m_run[n] = row_shift(m_run[n], l);
    if (quad == 0) {
      s_max[wave][16 * n + col] = m_run[n];
      s_sum[wave][16 * n + col] = l;
    }
  }
  // 16 threads a row, dims 4 c16 .. + 3 and 64 + 4 c16 .. + 3 each.
  const int r16 = tid >> 4, c16 = tid & 15;
  auto store = [&](int of_slot, int r, const float* acc, float l) TM_INLINED {
    const int at = (of_slot & (row_tiles - 1)) * kRows + r;
    const int t = by_group.token(at);
    if (pos0 + t < 0) return;  // before the request's first token: no row
    const int head = (head_group << head_shift) + (of_slot >> p.row_shift);
    float v_scale = 1.0f;
    if constexpr (kCache == CacheType::kE4m3) v_scale = p.value_scale[head];
    store_row<Type>(p.out + ((int64_t)(row0 + t) * p.heads + head * G + (at - t * G)) * kHeadDim, c16, acc,
                    inverse_sum(l), v_scale);
  };
  auto rows_of = [&](int of_slot) TM_INLINED { return min(kRows, part_rows - (of_slot & (row_tiles - 1)) * kRows); };
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    __syncthreads();
    if (16 * n >= min(kRows, part_rows)) break;
    float top = -INFINITY;
    for (int k = slot; k < kWaves; k += slots) top = fmaxf(top, s_max[k][16 * n + col]);
    // A row whose scores here are all -infinity: its weight is zero, and zero times an O that a NaN in V has
    // reached is NaN, as it must be (the compiler takes no number for NaN: it does not see which this one is).
    float weight = m_run[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[n] - top);
    asm volatile("" : "+v"(weight));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // dims 32 quad + 8 e + 4 half ..
        f32x4_t x;
#pragma unroll
        for (int m = 0; m < 4; ++m) x[m] = o[4 * half + m][n][e] * weight;
        const int chunk = (8 * quad + 2 * e + half) ^ col;
        *reinterpret_cast<f32x4_t*>(&o_lds[wave][col * kHeadDim + 4 * chunk]) = x;
      }
    }
    __syncthreads();
    const int slot_each = row_tiles > 1 ? 16 : min(16, part_rows - 16 * n);  // rows of a slot
    for (int i = r16; i < slots * slot_each; i += kThreads / 16) {
      const int of_slot = i / slot_each, at16 = i - of_slot * slot_each, r = 16 * n + at16;
      if (r >= rows_of(of_slot)) continue;
      float all = -INFINITY;
      for (int k = of_slot; k < kWaves; k += slots) all = fmaxf(all, s_max[k][r]);
      float l = 0.0f, acc[8] = {};
      for (int k = of_slot; k < kWaves; k += slots) {
        const float mk = s_max[k][r];
        l += mk == -INFINITY ? 0.0f : s_sum[k][r] * __builtin_amdgcn_exp2f(mk - all);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const f32x4_t x =
              *reinterpret_cast<const f32x4_t*>(&o_lds[k][at16 * kHeadDim + 4 * ((16 * half + c16) ^ at16)]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[4 * half + e] += x[e];
        }
      }
#pragma unroll
      for (int kind = 0; kind < 3; ++kind) {
        const unsigned* const odd = s_odd[of_slot * kRows + r][kind] + (c16 >> 3);
        // bits, and no number that is taken for finite
        float value = __uint_as_float(kind == 0 ? 0x7f800000u : kind == 1 ? 0xff800000u : 0x7fc00000u);
        asm volatile("" : "+v"(value));
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += odd[2 * (e >> 2)] >> (4 * (c16 & 7) + (e & 3)) & 1 ? value : 0.0f;
      }
      if (whole) {
        store(of_slot, r, acc, l);
      } else {
        const int row = of_slot * slot_rows + r;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const f32x4_t x = {acc[4 * half], acc[4 * half + 1], acc[4 * half + 2], acc[4 * half + 3]};
          group.store(share, row, 64 * half + 4 * c16, x);
        }
        if (c16 == 0) group.store_sums(share, row, all, l);
      }
    }
  }

  if (!whole) {
    merge_shares<kThreads, kFlight, kEach, true>(
        p, group, join, &s_last,
        [&](int row) TM_INLINED { return row % slot_rows < rows_of(row / slot_rows); },
        [&](int row, const float* acc, float l) TM_INLINED { store(row / slot_rows, row % slot_rows, acc, l); });
  }
}

template <class Type, CacheType kCache>
hipError_t launch_shape(const CachedParams& p, CachedShape shape, hipStream_t stream) {
  const dim3 grid((unsigned)p.workgroups), block(64 * shape.waves);
  if (shape.rows == 16 && shape.waves == 4) {
    hipLaunchKernelGGL((cached_attention_kernel<Type, kCache, 1, 4>), grid, block, 0, stream, p);
  } else if (shape.rows == 16 && shape.waves == 8) {
    hipLaunchKernelGGL((cached_attention_kernel<Type, kCache, 1, 8>), grid, block, 0, stream, p);
  } else if (shape.rows == 32 && shape.waves == 8) {
    hipLaunchKernelGGL((cached_attention_kernel<Type, kCache, 2, 8>), grid, block, 0, stream, p);
  } else {
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cached_attention(const CachedParams& p, CachedShape shape, bool fp16, CacheType cache,
                                   hipStream_t stream) {
  if (cache == CacheType::kE4m3) {
    return fp16 ? launch_shape<Fp16, CacheType::kE4m3>(p, shape, stream)
                : launch_shape<Bf16, CacheType::kE4m3>(p, shape, stream);
  }
  return fp16 ? launch_shape<Fp16, CacheType::kSame>(p, shape, stream)
              : launch_shape<Bf16, CacheType::kSame>(p, shape, stream);
}

}  // namespace tmx
