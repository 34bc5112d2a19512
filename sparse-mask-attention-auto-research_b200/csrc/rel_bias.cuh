// Learned bias by bucketed relative position, shared by the attention kernels
// that add it to their scores.
//
// The bias of query i and key j of head h is table[bucket(d)][h] with
// d = j - i - offset.  The buckets of one side are given by their smallest
// distances (`starts`, ascending from 0): the bucket of a distance is the
// last one that starts at or before it.  One-sided, a key at or after the
// query has distance 0; two-sided, keys after the query have `side` more
// buckets of their own.  The starts are whole numbers worked out on the host,
// so no bucket border depends on how a logarithm rounds.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sma_internal.h"

namespace sma {

__device__ __forceinline__ int bias_offset_of(const BiasSpec& s, int b) {
  if (s.offsets == nullptr) return s.offset;
  return max(-kMaxBiasOffset, min(kMaxBiasOffset, __ldg(s.offsets + b)));
}

// Bucket of relative position d; `starts` is the caller's copy of s.starts.
__device__ __forceinline__ int bias_bucket(const BiasSpec& s, const int* starts, int d) {
  const int far = s.two_sided ? (d < 0 ? -d : d) : (d < 0 ? -d : 0);
  int lo = 0, hi = s.side;  // starts[lo] <= far < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= far) lo = mid;
    else hi = mid;
  }
  return lo + ((s.two_sided && d > 0) ? s.side : 0);
}

// Where value i of a head's bias by relative position stands (bias_stride in
// sma_internal.h).
__device__ __forceinline__ int bias_at(int i) { return (i >> 2) * 16 + (i & 3); }

template <bool BF16>
__device__ __forceinline__ float bias_value(const BiasSpec& s, int bucket, int h) {
  const int64_t at = static_cast<int64_t>(bucket) * s.H + h;
  if constexpr (BF16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(s.table) + at));
  return __half2float(__ldg(static_cast<const __half*>(s.table) + at));
}

}  // namespace sma
