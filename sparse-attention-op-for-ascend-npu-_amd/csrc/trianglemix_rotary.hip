// Rotation of query and key rows by their positions, alone or with the write
// of the step's keys and values into a paged cache, for MI355X (gfx950).
//
// A pair of dims (a, b) of a head turns by the angle p f_i: (a cos - b sin,
// b cos + a sin).  The angle's turns p f_i / 2 pi are reduced to [-1/2, 1/2] in 64
// bits, where a position of 2^30 leaves 2^-24 of a turn; sine and cosine are
// taken of what is left in 32.
//
// A wave has eight heads of one token, a lane 16 dims of one of them: eight
// pairs, or 16 dims that are copied.  The wave forms the token's (at most 64)
// sines and cosines once, a frequency a lane, and hands them round through LDS.
// Query, key and value heads are numbered in a row, so that one launch serves all
// three and small head counts leave few lanes idle.
//
// Results go past the caches (non-temporal stores: 4096 tokens into an 8-bit cache
// 17.3 us, 18.5 with plain ones).
//
// What bounds it: memory for large chunks (8191 tokens of 40 heads 34.2 us, 4.9 TB/s as
// a library copy), the launch and two dependent round
// trips (position, then the rows' sines; the rows themselves are loaded beside
// them) for a decoding step.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "trianglemix_cached.h"
#include "trianglemix_device.h"

namespace tmx {
namespace {

constexpr int kRotateThreads = 256;
constexpr int kItems = kHeadDim / 16;  // of a head, one a lane
constexpr int kWaveHeads = 64 / kItems;

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

struct RotateBf16 { typedef bf16x8_t vec; typedef __bf16 elem; };
struct RotateFp16 { typedef f16x8_t vec; typedef _Float16 elem; };

// Eight numbers as e4m3 of their quotients by `scale`: ties to even, +-448 for
// what is larger, NaN for NaN.  The quotient is the product with the reciprocal and
// one step of its error, the division's rounding at a third of its instructions
// (4096 tokens: 17.3 us, with divisions 18.0); far beyond the range, where that step
// may overflow, the product alone says which end.  By scales below 2^-90 the numbers are
// divided: the error's step may be too small for a number of 32 bits there, and ties of
// such quotients would go astray.
__device__ __forceinline__ u32x2_t to_e4m3(const float* x, float scale) {
  const float reciprocal = 1.0f / scale;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float near = x[e] * reciprocal;
    const float step = __builtin_fmaf(__builtin_fmaf(-near, scale, x[e]), reciprocal, near);
    y[e] = fabsf(near) < 1024.0f ? __builtin_copysignf(step, near) : near;  // a zero keeps its sign
  }
  if (__builtin_expect(scale < 0x1p-90f, 0)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e] / scale;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if ((__float_as_uint(y[e]) & 0x7fffffffu) <= 0x7f800000u) y[e] = __builtin_amdgcn_fmed3f(y[e], -448.0f, 448.0f);
  }
  u32x2_t r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w], y[4 * w + 1], 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w + 2], y[4 * w + 3], v, true);
    r[w] = (unsigned)v;
  }
  return r;
}

template <class Type, bool kInterleaved, bool kCache, CacheType kStored>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(const RotateParams p, int waves_per_row) {
  __shared__ float2 turns[kRotateThreads / 64][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const unsigned id = blockIdx.x * (kRotateThreads / 64) + wave;
  const int row = (int)(id / (unsigned)waves_per_row);
  if (row >= p.rows) return;
  const int64_t position = p.positions[row];
  const int head = (int)(id % (unsigned)waves_per_row) * kWaveHeads + lane / kItems;
  const int item = lane % kItems;

  // This lane's 16 dims: a[e] and b[e] are pairs where they turn half by half.
  const int kind = head < p.heads ? 0 : head < p.heads + p.kv_heads ? 1 : head < p.heads + 2 * p.kv_heads ? 2 : 3;
  const int own = kind == 0 ? head : kind == 1 ? head - p.heads : head - p.heads - p.kv_heads;
  const bool turn = kind < 2 && 16 * item < p.rotary_dim;
  const int a_dim = !kInterleaved && turn ? 8 * item : 16 * item;
  const int b_dim = !kInterleaved && turn ? p.rotary_dim / 2 + 8 * item : 16 * item + 8;
  typename Type::vec raw_a = {}, raw_b = {};
  if (kind < 3) {
    const uint16_t* const from = (kind == 0 ? p.query + (int64_t)row * p.query_stride
                                  : kind == 1 ? p.key + (int64_t)row * p.key_stride
                                              : p.value + (int64_t)row * p.value_stride) + own * kHeadDim;
    raw_a = *reinterpret_cast<const typename Type::vec*>(from + a_dim);
    raw_b = *reinterpret_cast<const typename Type::vec*>(from + b_dim);
  }
  // What hangs on none of these is loaded beside them.
  const double frequency = p.frequencies[min(lane, p.rotary_dim / 2 - 1)];
  int64_t slot = -1;
  float scale = 1.0f;
  if constexpr (kCache) {
    slot = p.slots[row];
    if constexpr (kStored == CacheType::kE4m3) {
      if (kind == 1 || kind == 2) scale = (kind == 1 ? p.key_scale : p.value_scale)[own];
    }
  }
  if (position < 0) return;  // no row

  float2 mine = {1.0f, 0.0f};
  if (lane < p.rotary_dim / 2) {
    const double t = (double)position * (frequency * 0.15915494309189533577);
    const float half_turns = 2.0f * (float)(t - rint(t));
    float s, c;
    sincospif(half_turns, &s, &c);
    mine = {c * p.magnitude, s * p.magnitude};
  }
  turns[wave][lane] = mine;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own values: its LDS operations stay in order
  __builtin_amdgcn_wave_barrier();
  if (kind == 3) return;

  float a[8], b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    a[e] = (float)raw_a[e];
    b[e] = (float)raw_b[e];
  }
  if (turn) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 cs = turns[wave][8 * item + e];
      // pair e: dims e of both halves, or dims 2 e and 2 e + 1 of the 16
      float& x = !kInterleaved ? a[e] : e < 4 ? a[2 * e] : b[2 * e - 8];
      float& y = !kInterleaved ? b[e] : e < 4 ? a[2 * e + 1] : b[2 * e - 7];
      const float u = x, v = y;
      x = u * cs.x - v * cs.y;
      y = v * cs.x + u * cs.y;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      raw_a[e] = (typename Type::elem)a[e];
      raw_b[e] = (typename Type::elem)b[e];
    }
  }
  if (kind == 0) {
    uint16_t* const to = p.query_out + (int64_t)row * p.out_stride + own * kHeadDim;
    __builtin_nontemporal_store(raw_a, reinterpret_cast<typename Type::vec*>(to + a_dim));
    __builtin_nontemporal_store(raw_b, reinterpret_cast<typename Type::vec*>(to + b_dim));
    return;
  }
  if constexpr (kCache) {
    if (slot < 0 || slot >= p.num_slots) return;
    constexpr int kBytes = kStored == CacheType::kE4m3 ? 1 : 2;
    char* const to = (kind == 1 ? p.key_cache + slot / kPageSize * p.key_page_stride
                                : p.value_cache + slot / kPageSize * p.value_page_stride) +
                     (slot % kPageSize * p.kv_heads + own) * (kHeadDim * kBytes);
    if constexpr (kStored == CacheType::kE4m3) {
      __builtin_nontemporal_store(to_e4m3(a, scale), reinterpret_cast<u32x2_t*>(to + a_dim));
      __builtin_nontemporal_store(to_e4m3(b, scale), reinterpret_cast<u32x2_t*>(to + b_dim));
    } else {
      __builtin_nontemporal_store(raw_a, reinterpret_cast<typename Type::vec*>(to + 2 * a_dim));
      __builtin_nontemporal_store(raw_b, reinterpret_cast<typename Type::vec*>(to + 2 * b_dim));
    }
  }
}

template <class Type, bool kInterleaved>
hipError_t launch_type(const RotateParams& p, CacheType cache, hipStream_t stream) {
  const unsigned waves = (unsigned)(p.heads + 2 * p.kv_heads + kWaveHeads - 1) / kWaveHeads;
  const dim3 grid((unsigned)(((int64_t)p.rows * waves + kRotateThreads / 64 - 1) / (kRotateThreads / 64)));
  if (p.kv_heads == 0) {
    hipLaunchKernelGGL((rotate_kernel<Type, kInterleaved, false, CacheType::kSame>), grid, dim3(kRotateThreads), 0,
                       stream, p, (int)waves);
  } else if (cache == CacheType::kE4m3) {
    hipLaunchKernelGGL((rotate_kernel<Type, kInterleaved, true, CacheType::kE4m3>), grid, dim3(kRotateThreads), 0,
                       stream, p, (int)waves);
  } else {
    hipLaunchKernelGGL((rotate_kernel<Type, kInterleaved, true, CacheType::kSame>), grid, dim3(kRotateThreads), 0,
                       stream, p, (int)waves);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotate(const RotateParams& p, bool interleaved, bool fp16, CacheType cache, hipStream_t stream) {
  if (fp16) {
    return interleaved ? launch_type<RotateFp16, true>(p, cache, stream) : launch_type<RotateFp16, false>(p, cache, stream);
  }
  return interleaved ? launch_type<RotateBf16, true>(p, cache, stream) : launch_type<RotateBf16, false>(p, cache, stream);
}

}  // namespace tmx
