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

  __device__ __forceinline__ Shares(const CachedParams& p, int record_rows, int first_share, int share_step, int own,
                                    int shares)
      : record_bytes((unsigned)record_rows * ((kHeadDim + 2) * 4)), rows(record_rows), first(first_share),
        step(share_step), share(own), count(shares) {
    partials = __builtin_amdgcn_make_buffer_rsrc(
        (void*)p.partials, (short)0, shares > 1 ? (int)((unsigned)p.workgroups * record_bytes) : 0, kBufferFlags);
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

// Merges a shared group once its partials are stored: the workgroup that arrives last
// at a cluster of shares merges it, the one that arrives last of the clusters those
// (the same sums whichever they are).  16 threads a row, 8 dims each; where the rows
// leave threads over, `parts` of them share a row's partials and join through LDS.
// Eight partials' loads are in flight at a time.  held(row): whether the record's row
// is one; out(row, c8, acc, sum): its dims 8 c8 .. + 7.  Every thread calls it.
constexpr int kPartialsInFlight = 8;
template <int kThreads>
__device__ __forceinline__ int merge_parts(int rows) {
  int row_slots = 1;
  while (row_slots < rows && row_slots < kThreads / 16) row_slots *= 2;
  return kThreads / 16 / row_slots;
}
template <int kThreads, class Held, class Out>
__device__ __forceinline__ void merge_shares(const CachedParams& p, const Shares& shares, float (*join)[10], int* last,
                                             Held held, Out out) {
  const int tid = threadIdx.x, r16 = tid >> 4, c8 = tid & 15;
  const int parts = merge_parts<kThreads>(shares.rows), row_slots = kThreads / 16 / parts;
  const int cluster = kPartialsInFlight * parts, pg = r16 / row_slots;
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
    const int pg = r16 / row_slots;
    for (int rb = 0; rb < shares.rows; rb += row_slots) {
      const int row = rb + r16 % row_slots;
      const bool ok = row < shares.rows && held(row);
      float top = -INFINITY, l = 0.0f, acc[8] = {};
      if (ok) {
        for (int s0 = pg; s0 < count; s0 += kPartialsInFlight * parts) {
          float ms[kPartialsInFlight], ls[kPartialsInFlight];
          f32x4_t x[kPartialsInFlight][2];
#pragma unroll
          for (int j = 0; j < kPartialsInFlight; ++j) {
            // past the last one its loads fall outside the buffer's range
            const int s = s0 + j * parts;
            const unsigned at = s < count ? shares.record(from + s * stride) : kOutOfRange;
            ms[j] = __uint_as_float(
                __builtin_amdgcn_raw_buffer_load_b32(shares.partials, at + (shares.rows * kHeadDim + row) * 4, 0, kCpolAgent));
            ls[j] = __uint_as_float(
                __builtin_amdgcn_raw_buffer_load_b32(shares.partials, at + (shares.rows * (kHeadDim + 1) + row) * 4, 0, kCpolAgent));
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              x[j][half] = __builtin_bit_cast(
                  f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                               shares.partials, at + (row * kHeadDim + 8 * c8 + 4 * half) * 4, 0, kCpolAgent));
            }
          }
          float next = top;
#pragma unroll
          for (int j = 0; j < kPartialsInFlight; ++j) {
            if (s0 + j * parts >= count) ms[j] = -INFINITY;
            next = fmaxf(next, ms[j]);
          }
          const float shift = next == -INFINITY ? 0.0f : next;
          const float keep = __builtin_amdgcn_exp2f(top - shift);
          l *= keep;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] *= keep;
#pragma unroll
          for (int j = 0; j < kPartialsInFlight; ++j) {
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
        for (int e = 0; e < 8; ++e) join[tid][e] = acc[e];
        join[tid][8] = top;
        join[tid][9] = l;
        __syncthreads();
        if (pg == 0) {
          float all = top;
          for (int k = 1; k < parts; ++k) all = fmaxf(all, join[tid + k * 16 * row_slots][8]);
          const float shift = all == -INFINITY ? 0.0f : all;
          const float keep = __builtin_amdgcn_exp2f(top - shift);
          l *= keep;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] *= keep;
          for (int k = 1; k < parts; ++k) {
            const float* const other = join[tid + k * 16 * row_slots];
            const float w = __builtin_amdgcn_exp2f(other[8] - shift);
            l += other[9] * w;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += other[e] * w;
          }
          top = all;
        }
      } else if (!last_level) {
        __syncthreads();  // all have read the record that the result replaces
      }
      if (pg == 0 && ok) {
        if (last_level) {
          out(row, c8, acc, l);
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const f32x4_t x = {acc[4 * half], acc[4 * half + 1], acc[4 * half + 2], acc[4 * half + 3]};
            shares.store(from, row, 8 * c8 + 4 * half, x);
          }
          if (c8 == 0) shares.store_sums(from, row, top, l);
        }
      }
    }
    if (last_level) return;
  }
}

}  // namespace tmx

#endif  // TRIANGLEMIX_CACHED_DEVICE_H
