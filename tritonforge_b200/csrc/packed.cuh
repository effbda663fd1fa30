// Packed sequences: `S` sequences laid end to end in one token axis, offsets
// cu[0..S] (device int32, non-decreasing). Tokens before cu[0] or from cu[S] on
// are in no sequence.
#pragma once

#include "common.cuh"

namespace tf {

// The sequence that token t belongs to, if it is in one: the last s with cu[s] <= t
// (empty sequences own no token), in [0, S).
__device__ __forceinline__ int packed_sequence(const int* __restrict__ cu, int S, int64_t t) {
  int lo = 0, hi = S;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// An offset of cu, held inside [0, total] whatever the caller wrote there.
__device__ __forceinline__ int64_t packed_offset(const int* __restrict__ cu, int i, int64_t total) {
  const int64_t v = cu[i];
  return v < 0 ? 0 : (v > total ? total : v);
}

}  // namespace tf
