// Attention of chunks of query rows over a request's paged cache, of e4m3 numbers
// or of the queries' own 16-bit type, for MI355X (gfx950): the rows that are too many
// for trianglemix_cached.hip.
//
// A workgroup is eight waves of 32 rows over the same keys: 256 rows of a (request, KV
// head), all heads of the GQA group times consecutive tokens, rows numbered token *
// G + head.  A step is 64 keys.  Each goes from memory into registers a step ahead,
// becomes 16-bit numbers there (e4m3: K of the queries' type, V fp16 with fp16
// weights, both exact) and is written to LDS for all waves while the matrix cores work
// at the step before's scores: once for 256 rows, where waves that load their operands
// themselves convert them for each 32 or 64 (2048 rows of 32749 tokens: 1450 us so).
// Two slots of 32 KB; one barrier a step.  Where 256 rows a workgroup leave CUs idle, a
// workgroup has 128 rows and its waves one tile of a step each (two key parts, joined in
// LDS at the end).
//
// Contractions (per wave, 32-key tiles x 32 rows, v_mfma_f32_32x32x16)
//   S^T (keys x rows) = K Q^T     A = K rows from LDS, B = Q in registers
//   O^T (dims x rows) += V^T P^T  A = V by ds_read_b64_tr_b16, B = P
// with the operand layouts of trianglemix_device.h.
//
// What bounds it: 2048 rows of 32749 tokens, 32 heads, 1035 us, 1030 TFLOP/s, where a
// library product of 8192^3 reaches 1205: power, the clock is 2.1 of 2.4 GHz.  A
// step takes 4300 cycles; MFMAs are busy 47 % of them, LDS 36 %, and the seven vector
// instructions to an MFMA (exponentials, sums, conversions) about as long as the
// MFMAs.  Waves half a step apart, so that one's exponentials run beside the other's
// products, take the same time.  512 rows of 8192 tokens: 85 us, 71 of them in the
// loop, the rest start, partials of four shares a part (34 MB) and their merge.
//
// Parts whose keys are shared by several workgroups (few rows, many keys) are merged
// as in trianglemix_cached_device.h.  Numerics as in trianglemix_cached.hip.  V entries
// that are no finite numbers never enter a product: they are noted, on their way to
// LDS, for the rows that attend them.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_cached_device.h"

namespace tmx {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kStepKeys = 64;
constexpr int kSlotBytes = kStepKeys * kRowBytes;  // 16 KB: K or V of one step
static_assert(kWaves * 32 == kChunkRows && kPageSize % kStepKeys == 0, "a step stays inside a page");
static_assert(kStepKeys == 2 * kKvTile, "a tile for each of two key parts");

// What a thread carries of a step: 16 numbers of K and of V.
template <class Type, CacheType kCache>
struct Staged;

template <class Type>
struct Staged<Type, CacheType::kSame> {
  typedef Type Weight;
  static constexpr int kElemBytes = 2;
  u32x4_t k[2], v[2];  // rows tid / 16 and 32 + tid / 16, chunk tid % 16

  static __device__ __forceinline__ int row(int half) { return 32 * half + (int)(threadIdx.x >> 4); }
  static __device__ __forceinline__ int chunk(int) { return threadIdx.x & 15; }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, int token_bytes) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = row(half) * token_bytes + 16 * chunk(half);
      k[half] = __builtin_amdgcn_raw_buffer_load_b128(kr, at, 0, 0);
      v[half] = __builtin_amdgcn_raw_buffer_load_b128(vr, at, 0, 0);
    }
  }
  __device__ __forceinline__ u32x4_t key_chunk(int half) const { return k[half]; }
  __device__ __forceinline__ u32x4_t value_chunk(int half) const { return v[half]; }
  // Whether some V number is not finite: a carry out of its exponent's place.
  __device__ __forceinline__ bool odd_value() const {
    unsigned odd = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) odd |= (v[e >> 2][e & 3] & 0x7fff7fffu) + (0x8000u - Type::kExp) * 0x10001u;
    return (odd & 0x80008000u) != 0;
  }
};

template <class Type>
struct Staged<Type, CacheType::kE4m3> {
  typedef Fp16 Weight;
  static constexpr int kElemBytes = 1;
  u32x4_t k, v;  // row tid / 8, chunks 2 (tid % 8) and the next

  static __device__ __forceinline__ int row(int) { return threadIdx.x >> 3; }
  static __device__ __forceinline__ int chunk(int half) { return 2 * (threadIdx.x & 7) + half; }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, int token_bytes) {
    const int at = row(0) * token_bytes + 16 * (threadIdx.x & 7);
    k = __builtin_amdgcn_raw_buffer_load_b128(kr, at, 0, 0);
    v = __builtin_amdgcn_raw_buffer_load_b128(vr, at, 0, 0);
  }
  template <class To>
  static __device__ __forceinline__ u32x4_t widened(u32x4_t x, int half) {
    return u32x4_t{from_e4m3<To, false>(x[2 * half]), from_e4m3<To, true>(x[2 * half]),
                   from_e4m3<To, false>(x[2 * half + 1]), from_e4m3<To, true>(x[2 * half + 1])};
  }
  __device__ __forceinline__ u32x4_t key_chunk(int half) const { return widened<Type>(k, half); }
  __device__ __forceinline__ u32x4_t value_chunk(int half) const { return widened<Fp16>(v, half); }
  __device__ __forceinline__ bool odd_value() const {
    unsigned odd = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= (v[e] & 0x7f7f7f7fu) + 0x01010101u;
    return (odd & 0x80808080u) != 0;
  }
};

template <class Type, CacheType kCache, int kKeyParts>
__global__ void __launch_bounds__(kThreads, 1) cached_chunk_kernel(const CachedParams p) {
  constexpr int kRowTiles = kWaves / kKeyParts, kRows = 32 * kRowTiles, kTiles = 2 / kKeyParts;  // a wave's tiles of a step
  typedef Staged<Type, kCache> Stage;
  typedef typename Stage::Weight Weight;
  typedef typename Type::elem elem;
  constexpr int kHeadBytes = kHeadDim * Stage::kElemBytes;
  constexpr float kWeightBits = std::is_same_v<Weight, Fp16> ? 7.0f : 0.0f;

  __shared__ __attribute__((aligned(1024))) char kv_lds[4 * kSlotBytes];
  char* const k_lds = kv_lds;
  char* const v_lds = kv_lds + 2 * kSlotBytes;
  __shared__ unsigned s_odd[kRows][3][4];  // note_odd: a bit a dim, for +infinity, -infinity, NaN
  __shared__ float s_max[kWaves][32], s_sum[kWaves][32];
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int n = lane & 31, half = lane >> 5;  // row of the wave's tile
  const int G = p.group;
  const GroupDivider by_group(p.group);
  const int token_bytes = p.kv_heads * kHeadBytes;

  // ---- the part, and this workgroup's share of its steps ----
  unsigned id = blockIdx.x;
  const int kv_head = (int)(id % (unsigned)p.kv_heads);  // of one XCD where there are eight: it shares their keys
  id /= (unsigned)p.kv_heads;
  // The first p.full_parts parts (of all requests) have a workgroup a KV head, the others p.splits.
  int splits = 1, share = 0;
  if ((int)id >= p.full_parts) {
    splits = p.splits;
    id -= (unsigned)p.full_parts;
    share = (int)(id % (unsigned)splits);
    id = id / (unsigned)splits + (unsigned)p.full_parts;
  }
  const int request = (int)(id % (unsigned)p.batch);
  const int part = p.row_parts - 1 - (int)(id / (unsigned)p.batch);  // later rows attend more keys
  const int len = max(p.seq_lens[request], 0);
  const int part_tokens = min(p.part_tokens, p.rows - part * p.part_tokens);
  const int part_rows = part_tokens * G;
  const int pos0 = len - p.rows + part * p.part_tokens;  // of the part's first token; a negative one is no row
  const Tiles<kStepKeys> tiles(p, pos0, pos0 + part_tokens - 1);
  if (tiles.count == 0) return;
  const int each = max((tiles.count + splits - 1) / splits, kLeastSteps), shares = (tiles.count + each - 1) / each;
  if (share >= shares) return;
  const int lo = share * each, steps = min(each, tiles.count - lo);
  const int unshared = p.full_parts * p.kv_heads;  // workgroups without records
  const Shares group(p, p.workgroups - unshared, min(kRows, p.part_tokens * G),
                     (int)blockIdx.x - unshared - share * p.kv_heads, p.kv_heads, share, shares);
  const int tokens = min(len, p.table_cols * kPageSize);  // with a key
  const int row0 = request * p.rows + part * p.part_tokens;  // of query and out
  for (int i = tid; i < kRows * 12; i += kThreads) (&s_odd[0][0][0])[i] = 0;

  // ---- this wave's rows, and its part of a step's keys ----
  const int key_part = wave / kRowTiles;
  const int row_base = 32 * (wave % kRowTiles), row = row_base + n;
  const int valid_rows = min(32, part_rows - row_base);  // none: the wave only loads
  const int token = by_group.token(row);
  const bool ok = n < valid_rows;
  const int row_pos = ok ? pos0 + token : -1;
  const int first_pos = pos0 + by_group.token(row_base);
  const int last_pos = valid_rows > 0 ? pos0 + by_group.token(row_base + valid_rows - 1) : -1;
  const int low = p.window < 0 ? 0 : max(row_pos, 0) - p.window;  // the first key of the row's window,
  const int last_low = p.window < 0 ? 0 : max(last_pos, 0) - p.window;  // the last row's
  const int first_low = p.window < 0 ? 0 : max(first_pos, 0) - p.window;
  i16x8_t q[8];
  {
    const uint16_t* const from =
        p.query + (int64_t)(row0 + token) * p.query_stride + (int64_t)(kv_head * G + (row - token * G)) * kHeadDim;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      q[c] = i16x8_t{};
      if (ok) q[c] = *reinterpret_cast<const i16x8_t*>(from + 16 * c + 8 * half);
    }
  }
  float c2 = p.scale_log2, v_scale = 1.0f;
  if constexpr (kCache == CacheType::kE4m3) {
    c2 *= p.key_scale[kv_head];
    v_scale = p.value_scale[kv_head];
  }

  // ---- steps ----
  const ConstInts table = (ConstInts)(p.block_table + (int64_t)request * p.table_stride);
  auto first_key = [&](int i) TM_INLINED { return tiles.tile(lo + i) * kStepKeys; };
  auto entry = [&](int i) TM_INLINED {  // page of the cache, or -1
    int phys = -1;
    const int t = tiles.tile(lo + i);
    if (i < steps && t < tiles.end) phys = table[t / (kPageSize / kStepKeys)];
    return (unsigned)phys < (unsigned)p.num_pages ? phys : -1;
  };
  Stage stage;
  auto load = [&](int i, int phys) TM_INLINED {
    const int key0 = first_key(i);
    const int valid = phys < 0 ? 0 : min(kStepKeys, tokens - key0);
    const int range = valid > 0 ? (valid - 1) * token_bytes + kHeadBytes : 0;
    const int64_t in_page = kv_head * kHeadBytes + (int64_t)(key0 % kPageSize) * token_bytes;
    stage.load(__builtin_amdgcn_make_buffer_rsrc((void*)(p.key_cache + max(phys, 0) * p.key_page_stride + in_page), (short)0,
                                                 range, kBufferFlags),
               __builtin_amdgcn_make_buffer_rsrc((void*)(p.value_cache + max(phys, 0) * p.value_page_stride + in_page),
                                                 (short)0, range, kBufferFlags),
               token_bytes);
  };
  // Notes the numbers of a V chunk that are not finite for the rows that attend their key.
  auto note_odd = [&](int key0, int r, int chunk, const u32x4_t& x) TM_INLINED {
    unsigned kinds[3] = {};  // of the chunk's eight dims
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int kind = 1; kind < 4; ++kind) {
        kinds[kind - 1] |= (only_kind<Weight>(x[e], kind) ? 1u : 0u) << (2 * e) |
                           (only_kind<Weight>(x[e] >> 16, kind) ? 2u : 0u) << (2 * e);
      }
    }
    unsigned long long left = __ballot((kinds[0] | kinds[1] | kinds[2]) != 0);
    while (left) {
      const int from = __ffsll(left) - 1;
      left &= left - 1;
      const int key = key0 + __builtin_amdgcn_readlane(r, from), at = __builtin_amdgcn_readlane(chunk, from);
      unsigned bits[3];
#pragma unroll
      for (int kind = 0; kind < 3; ++kind) {
        bits[kind] = (unsigned)__builtin_amdgcn_readlane((int)kinds[kind], from) << (8 * (at & 3));
      }
      for (int row = lane; row < part_rows; row += 64) {
        const int pos = pos0 + by_group.token(row);
        if (key <= pos && (p.window < 0 || key >= max(pos, 0) - p.window || key < p.sinks)) {
#pragma unroll
          for (int kind = 0; kind < 3; ++kind) atomicOr(&s_odd[row][kind][at >> 2], bits[kind]);
        }
      }
    }
  };
  auto write = [&](int i) TM_INLINED {  // the staged step into its slot
    char* const ks = k_lds + (i & 1) * kSlotBytes;
    char* const vs = v_lds + (i & 1) * kSlotBytes;
    const bool odd = __builtin_expect(__any(stage.odd_value()), 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = Stage::row(h), chunk = Stage::chunk(h);
      *reinterpret_cast<u32x4_t*>(ks + r * kRowBytes + 16 * k_slot(r, chunk)) = stage.key_chunk(h);
      u32x4_t x = stage.value_chunk(h);
      if (odd) {
        note_odd(first_key(i), r, chunk, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = only_kind<Weight>(x[e], 0) | only_kind<Weight>(x[e] >> 16, 0) << 16;
      }
      *reinterpret_cast<u32x4_t*>(vs + r * kRowBytes + 16 * v_slot(r, chunk)) = x;
    }
  };

  float m_run = -INFINITY, l_run = 0.0f;  // of the row; the sum over this lane's keys
  f32x16_t o[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) o[m] = f32x16_t{};
  const int k_off = n * kRowBytes + 16 * k_slot(n, half);
  const int v_key = 4 * half + ((lane & 15) >> 2), v_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const int v_off = v_key * kRowBytes + 16 * v_slot(v_key, v_dim >> 3) + 2 * (v_dim & 7);

  auto active = [&](int i, int phys) TM_INLINED {  // whether some row of the wave attends some key of the step
    const int key0 = first_key(i);
    return phys >= 0 && key0 <= last_pos && (key0 + kStepKeys - 1 >= first_low || key0 < p.sinks);
  };
  f32x16_t s[kTiles];
  auto scores = [&](int i) TM_INLINED {
    const char* const ks = k_lds + (i & 1) * kSlotBytes;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) s[t] = f32x16_t{};
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const i16x8_t a = *reinterpret_cast<const i16x8_t*>(ks + (t + key_part) * kTileBytes + (k_off ^ (32 * c)));
        s[t] = Type::mfma32(a, q[c], s[t]);
      }
    }
  };
  auto values = [&](int i) TM_INLINED {
    const int key0 = first_key(i);
    const char* const vs = v_lds + (i & 1) * kSlotBytes;
    if (key0 + kStepKeys - 1 > first_pos || (key0 < last_low && key0 + kStepKeys - 1 >= p.sinks)) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int key = key0 + 32 * (t + key_part) + elem_key(v) + 4 * half;
          s[t][v] = key <= row_pos && (key >= low || key < p.sinks) ? s[t][v] : -INFINITY;
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < 16; ++v) top = fmaxf(top, fmaxf(s[0][v], s[kTiles - 1][v]));
    top = half_max(top) * c2;
    if (__any(top > m_run + kLazyRescale)) {
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int m = 0; m < 4; ++m) o[m] *= alpha;
      m_run = m_new;
    }
    const float shift = kWeightBits - (m_run == -INFINITY ? 0.0f : m_run);
    i16x8_t pb[2 * kTiles];
    float add = 0.0f;
#pragma unroll
    for (int j = 0; j < 2 * kTiles; ++j) {
      typename Weight::vec weight;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 1][8 * (j & 1) + e], c2, shift));
        add += x;
        weight[e] = (typename Weight::elem)x;
      }
      pb[j] = __builtin_bit_cast(i16x8_t, weight);
    }
    l_run += add;
#pragma unroll
    for (int j = 0; j < 2 * kTiles; ++j) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const char* const at = vs + (16 * j + 32 * key_part) * kRowBytes + (v_off ^ (64 * m));
        const i16x4_t lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(at));
        const i16x4_t hi4 =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(at + 8 * kRowBytes));
        o[m] = Weight::mfma32(__builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7), pb[j], o[m]);
      }
    }
  };

  // Step i + 1 is staged when step i begins and is written while the matrix cores work
  // at its scores; step i + 2 is loaded from then on.
  int phys = entry(0), next = entry(1), behind = entry(2);
  load(0, phys);
  __syncthreads();  // s_odd is clear
  write(0);
  load(1, next);
  __syncthreads();
  for (int i = 0; i < steps; ++i) {
    const bool on = active(i, phys);
    if (on) scores(i);
    __builtin_amdgcn_sched_barrier(0);
    if (i + 1 < steps) write(i + 1);
    load(i + 2, behind);
    phys = next;
    next = behind;
    behind = entry(i + 3);
    __builtin_amdgcn_sched_barrier(0);
    if (on) values(i);
    __syncthreads();
  }

  // ---- results: this lane's row, dims 32 m + 8 v + 4 half .. + 3 ----
  float l = half_sum(l_run);
  m_run = row_shift(m_run, l);
  if constexpr (kKeyParts == 2) {
    // the second key part's sums, register by register, to the waves that have the first
    float* const parts = reinterpret_cast<float*>(kv_lds) + (row_base / 32) * (64 * 64) + lane;
    static_assert(kRowTiles * 64 * 64 * 4 <= 4 * kSlotBytes, "they fit the slots");
    if (half == 0) {
      s_max[wave][n] = m_run;
      s_sum[wave][n] = l;
    }
    __syncthreads();
    const int other = wave ^ kRowTiles;
    const float top = fmaxf(m_run, s_max[other][n]);
    const float keep = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - top);
    if (key_part == 1) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
#pragma unroll
        for (int v = 0; v < 16; ++v) parts[64 * (16 * m + v)] = m_run == -INFINITY ? 0.0f : o[m][v] * keep;
      }
    }
    __syncthreads();
    if (key_part == 0) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          o[m][v] = (m_run == -INFINITY ? 0.0f : o[m][v] * keep) + parts[64 * (16 * m + v)];
        }
      }
      const float theirs = s_max[other][n];
      l = (m_run == -INFINITY ? 0.0f : l * keep) +
          (theirs == -INFINITY ? 0.0f : s_sum[other][n] * __builtin_amdgcn_exp2f(theirs - top));
      m_run = top;
    }
  }
#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int kind = 0; kind < 3; ++kind) {
      const unsigned odd = s_odd[row][kind][m] >> (4 * half);
      float value = __uint_as_float(kind == 0 ? 0x7f800000u : kind == 1 ? 0xff800000u : 0x7fc00000u);
      asm volatile("" : "+v"(value));  // bits, and no number that is taken for finite
#pragma unroll
      for (int v = 0; v < 16; ++v) o[m][v] += odd >> elem_key(v) & 1 ? value : 0.0f;
    }
  }
  auto out_row = [&](int r) TM_INLINED {
    const int t = by_group.token(r);
    return p.out + ((int64_t)(row0 + t) * p.heads + kv_head * G + (r - t * G)) * kHeadDim;
  };
  // 64 dims at a time through the wave's part of LDS, so that a store's lanes lie side by
  // side, 256 bytes of a row.
  if (key_part == 0) {
    const float inverse = shares > 1 ? 1.0f : inverse_sum(l), scale = shares > 1 ? 1.0f : v_scale;
    char* const own = kv_lds + (row_base / 32) * (4 * kSlotBytes / kRowTiles);
    static_assert(32 * 64 * 4 <= 4 * kSlotBytes / kWaves, "64 dims of 32 rows fit it");
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own values: its LDS operations stay in order
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
      for (int c = 0; c < 16; c += 2) {  // dims 4 (c + half) .. + 3 of the 64
        const int m = 2 * side + (c >> 3), v = 4 * ((c & 7) >> 1);
        *reinterpret_cast<f32x4_t*>(own + 256 * n + 16 * ((c + half) ^ (n & 15))) =
            f32x4_t{o[m][v] * inverse * scale, o[m][v + 1] * inverse * scale, o[m][v + 2] * inverse * scale,
                    o[m][v + 3] * inverse * scale};
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 4), c = lane & 15;
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(own + 256 * r + 16 * (c ^ (r & 15)));
        if (r >= valid_rows) continue;
        if (shares > 1) {
          group.store(share, row_base + r, 64 * side + 4 * c, x);
        } else if (pos0 + by_group.token(row_base + r) >= 0) {  // else before the request's first token: no row
          typedef elem vec4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<vec4*>(out_row(row_base + r) + 64 * side + 4 * c) = __builtin_convertvector(x, vec4);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (shares > 1 && ok && half == 0) group.store_sums(share, row, m_run, l);
  }
  if (shares == 1) return;
  static_assert(kChunkRows / 2 - (kMaxGroup - 1) >= kThreads / 16, "a record's rows leave no thread over to join");
  merge_shares<kThreads, 4, 2, false>(
      p, group, nullptr, &s_last, [&](int r) TM_INLINED { return r < part_rows; },
      [&](int r, const float* acc, float sum) TM_INLINED {
        if (pos0 + by_group.token(r) >= 0) store_row<Type>(out_row(r), tid & 15, acc, inverse_sum(sum), v_scale);
      });
}

template <class Type, CacheType kCache>
hipError_t launch_rows(const CachedParams& p, int rows, hipStream_t stream) {
  const dim3 grid((unsigned)p.workgroups), block(kThreads);
  if (rows == kChunkRows) {
    hipLaunchKernelGGL((cached_chunk_kernel<Type, kCache, 1>), grid, block, 0, stream, p);
  } else {
    hipLaunchKernelGGL((cached_chunk_kernel<Type, kCache, 2>), grid, block, 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cached_chunks(const CachedParams& p, int rows, bool fp16, CacheType cache, hipStream_t stream) {
  if (cache == CacheType::kE4m3) {
    return fp16 ? launch_rows<Fp16, CacheType::kE4m3>(p, rows, stream) : launch_rows<Bf16, CacheType::kE4m3>(p, rows, stream);
  }
  return fp16 ? launch_rows<Fp16, CacheType::kSame>(p, rows, stream) : launch_rows<Bf16, CacheType::kSame>(p, rows, stream);
}

}  // namespace tmx
