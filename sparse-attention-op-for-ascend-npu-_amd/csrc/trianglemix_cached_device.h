// Device code that the kernels of attention over a cache share
// (trianglemix_cached.hip, trianglemix_chunks.hip): the keys that rows may attend,
// 16-bit numbers of 8-bit ones, and the merge of groups that are shared out.
#ifndef TRIANGLEMIX_CACHED_DEVICE_H
#define TRIANGLEMIX_CACHED_DEVICE_H

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "trianglemix_cached.h"
#include "trianglemix_lists.h"

namespace tmx {

#define TM_INLINED __attribute__((always_inline))  // a call would put all that a lambda names into memory

typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));

typedef const __attribute__((address_space(4))) int32_t* ConstInts;  // read by scalar loads

// The bits of two 16-bit numbers of type Type from two e4m3 ones.
template <class Type, bool kHigh>
__device__ __forceinline__ unsigned from_e4m3(unsigned x) {
  if constexpr (std::is_same_v<Type, Fp16>) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, kHigh));
  } else {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, kHigh));
  }
}

// The tiles of kKeys keys that rows at first_pos .. last_pos may attend: `sinks` from
// the first on, then first .. end - 1; at least one where there is a row.
template <int kKeys>
struct Tiles {
  int sinks, first, end, count;
  __device__ __forceinline__ Tiles(const CachedParams& p, int first_pos, int last_pos) {
    end = (min(max(last_pos, -1) + 1, p.table_cols * kPageSize) + kKeys - 1) / kKeys;
    const int first_key = p.window < 0 ? 0 : max(0, max(0, first_pos) - p.window);
    first = min(first_key / kKeys, end);
    sinks = min((int)(((unsigned)p.sinks + kKeys - 1) / kKeys), first);
    count = last_pos < 0 ? 0 : max(1, sinks + end - first);
  }
  __device__ __forceinline__ int tile(int i) const { return i < sinks ? i : first + (i - sinks); }
};

// Partials of a group that several workgroups share: record s of the group is that
// of the workgroup that has share s, the O of `rows` rows, then their row maxima and
// sums; its arrival words are those of the shares' workgroups.
struct Shares {
  __amdgpu_buffer_rsrc_t partials;
  unsigned record_bytes;
  int rows;         // of a record
  int first, step;  // workgroup of share 0, and from one share to the next
  int share, count;

  __device__ __forceinline__ Shares(const CachedParams& p, int records, int record_rows, int first_share, int share_step,
                                    int own, int shares)
      : record_bytes((unsigned)record_rows * ((kHeadDim + 2) * 4)), rows(record_rows), first(first_share),
        step(share_step), share(own), count(shares) {
    partials = __builtin_amdgcn_make_buffer_rsrc(
        (void*)p.partials, (short)0, shares > 1 ? (int)((unsigned)records * record_bytes) : 0, kBufferFlags);
  }
  __device__ __forceinline__ unsigned record(int s) const { return (unsigned)(first + s * step) * record_bytes; }
  // Four dims of a row of record s; its maximum and sum.
  __device__ __forceinline__ void store(int s, int row, int dim, f32x4_t x) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), partials,
                                           record(s) + (unsigned)(row * kHeadDim + dim) * 4, 0, kCpolAgent);
  }
  __device__ __forceinline__ void store_sums(int s, int row, float max, float sum) const {
    const unsigned at = record(s) + (unsigned)(rows * kHeadDim + row) * 4;
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(max), partials, at, 0, kCpolAgent);
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(sum), partials, at + (unsigned)rows * 4, 0, kCpolAgent);
  }
};

// What a row's numbers are multiplied by, of their weights' sum: a NaN sum fails the comparison, and must reach the
// result.  The values' scale is a factor of its own: in one with a small scale a large sum would leave no bits
// (scales go down to 2^-126, sums of fp16 weights up to 2^28 and more).
__device__ __forceinline__ float inverse_sum(float sum) {
  return (__float_as_uint(sum) & 0x7fffffffu) > 0x7f800000u ? sum : sum > 0.0f ? 1.0f / sum : 0.0f;
}

// A row's numbers of the thread c16 of its 16, as merge_shares has them, times the two factors.
template <class Type>
__device__ __forceinline__ void store_row(uint16_t* row, int c16, const float* acc, float inverse, float scale) {
  typedef typename Type::elem vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    vec4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (typename Type::elem)(acc[4 * half + e] * inverse * scale);
    *reinterpret_cast<vec4*>(row + 64 * half + 4 * c16) = y;
  }
}

// Merges a shared group once its partials are stored: the workgroup that arrives last
// at a cluster of shares merges it, the one that arrives last of the clusters those
// (the same sums whichever they are).  16 threads a row, dims 4 c16 .. + 3 and 64 + 4
// c16 .. + 3 each (what they load or store at once lies side by side); where the rows
// leave threads over, `parts` of them share a row's partials and join through LDS (kJoin;
// without it they never are, and `join` is null).  A thread has the loads of kFlight
// partials of kEach rows in flight.  held(row): whether the record's row is one; out(row,
// acc, sum): the thread's dims of it.  Every thread calls it.
template <int kThreads>
__device__ __forceinline__ int merge_parts(int rows) {
  int row_slots = 1;
  while (row_slots < rows && row_slots < kThreads / 16) row_slots *= 2;
  return kThreads / 16 / row_slots;
}
template <int kThreads, int kFlight, int kEach, bool kJoin, class Held, class Out>
__device__ __forceinline__ void merge_shares(const CachedParams& p, const Shares& shares, float (*join)[10], int* last,
                                             Held held, Out out) {
  const int tid = threadIdx.x, r16 = tid >> 4, c16 = tid & 15;
  const int parts = kJoin ? merge_parts<kThreads>(shares.rows) : 1, row_slots = kThreads / 16 / parts;
  const int cluster = kFlight * parts, pg = r16 / row_slots;
  for (int level = 0; level < 2; ++level) {
    // the shares that are merged: `count` from `from` on, every stride-th
    const int stride = level == 0 ? 1 : cluster;
    const int from = level == 0 ? shares.share / cluster * cluster : 0;
    const int count = level == 0 ? min(cluster, shares.count - from) : (shares.count + cluster - 1) / cluster;
    const bool last_level = level == 1 || shares.count <= cluster;
    wait_dma();  // this wave's partial stores have completed
    __syncthreads();
    // words: the cluster's first share's; the group's second share's
    unsigned long long* const word = p.counters + shares.first + (level == 0 ? from : 1) * shares.step;
    if (tid == 0) {
      *last = (int)(count_arrival(word, p.epoch) == (unsigned long long)count);
      // The word is left at this launch's tag with a count of zero for the next one.
      if (*last) __hip_atomic_store(word, p.epoch << kEpochShift, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return;
    for (int rb = 0; rb < shares.rows; rb += kEach * row_slots) {
      float top[kEach], l[kEach], acc[kEach][8];
      int row[kEach];
      bool ok[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        row[i] = rb + i * row_slots + r16 % row_slots;
        ok[i] = row[i] < shares.rows && held(row[i]);
        top[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[i][e] = 0.0f;
      }
      for (int s0 = pg; s0 < count; s0 += kFlight * parts) {
        float ms[kEach][kFlight], ls[kEach][kFlight];
        f32x4_t x[kEach][kFlight][2];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
#pragma unroll
          for (int j = 0; j < kFlight; ++j) {
            // past the last one, and of what is no row, its loads fall outside the buffer's range
            const int s = s0 + j * parts;
            const unsigned at = s < count && ok[i] ? shares.record(from + s * stride) : kOutOfRange;
            ms[i][j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                shares.partials, at + (shares.rows * kHeadDim + row[i]) * 4, 0, kCpolAgent));
            ls[i][j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                shares.partials, at + (shares.rows * (kHeadDim + 1) + row[i]) * 4, 0, kCpolAgent));
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              x[i][j][half] = __builtin_bit_cast(
                  f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                               shares.partials, at + (row[i] * kHeadDim + 64 * half + 4 * c16) * 4, 0, kCpolAgent));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          float next = top[i];
#pragma unroll
          for (int j = 0; j < kFlight; ++j) {
            if (s0 + j * parts >= count) ms[i][j] = -INFINITY;
            next = fmaxf(next, ms[i][j]);
          }
          const float shift = next == -INFINITY ? 0.0f : next;
          const float keep = __builtin_amdgcn_exp2f(top[i] - shift);
          l[i] *= keep;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[i][e] *= keep;
#pragma unroll
          for (int j = 0; j < kFlight; ++j) {
            const float w = __builtin_amdgcn_exp2f(ms[i][j] - shift);
            l[i] += ls[i][j] * w;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[i][e] += x[i][j][e >> 2][e & 3] * w;
          }
          top[i] = next;
        }
      }
      if (parts > 1) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          __syncthreads();
#pragma unroll
          for (int e = 0; e < 8; ++e) join[tid][e] = acc[i][e];
          join[tid][8] = top[i];
          join[tid][9] = l[i];
          __syncthreads();
          if (pg == 0) {
            float all = top[i];
            for (int k = 1; k < parts; ++k) all = fmaxf(all, join[tid + k * 16 * row_slots][8]);
            const float shift = all == -INFINITY ? 0.0f : all;
            const float keep = __builtin_amdgcn_exp2f(top[i] - shift);
            l[i] *= keep;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[i][e] *= keep;
            for (int k = 1; k < parts; ++k) {
              const float* const other = join[tid + k * 16 * row_slots];
              const float w = __builtin_amdgcn_exp2f(other[8] - shift);
              l[i] += other[9] * w;
#pragma unroll
              for (int e = 0; e < 8; ++e) acc[i][e] += other[e] * w;
            }
            top[i] = all;
          }
        }
      } else if (!last_level) {
        __syncthreads();  // all have read the records that the results replace
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (pg != 0 || !ok[i]) continue;
        if (last_level) {
          out(row[i], acc[i], l[i]);
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const f32x4_t x = {acc[i][4 * half], acc[i][4 * half + 1], acc[i][4 * half + 2], acc[i][4 * half + 3]};
            shares.store(from, row[i], 64 * half + 4 * c16, x);
          }
          if (c16 == 0) shares.store_sums(from, row[i], top[i], l[i]);
        }
      }
    }
    if (last_level) return;
  }
}

}  // namespace tmx

#endif  // TRIANGLEMIX_CACHED_DEVICE_H
