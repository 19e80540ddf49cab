// Device helpers shared by the kernels on the paged key/value cache.
#pragma once

#include <cstdint>

#include "ptx.cuh"

namespace dtb {

// New tokens of sequence b, clamped to the tensor whatever query_start holds.
__device__ __forceinline__ int2 new_rows(const int32_t* query_start, int b, int T) {
  const int lo = min(max(__ldg(query_start + b), 0), T);
  const int hi = min(max(__ldg(query_start + b + 1), lo), T);
  return make_int2(lo, hi);
}

// Sequence of token t: the last b with query_start[b] <= t, or -1 where t belongs to none.  query_start ascends.
__device__ __forceinline__ int sequence_of(const int32_t* query_start, int B, int t) {
  int lo = 0, hi = B;                      // invariant: query_start[lo - 1] <= t < query_start[hi + 1], where those exist
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(query_start + mid) <= t) lo = mid; else hi = mid - 1;
  }
  return lo < B && __ldg(query_start + lo) <= t && t < __ldg(query_start + lo + 1) ? lo : -1;
}

// Tokens of a sequence that its row of the page table can name.
__device__ __forceinline__ int table_len(const int32_t* kv_len, int b, int64_t capacity) {
  return static_cast<int>(min(static_cast<int64_t>(max(__ldg(kv_len + b), 0)), capacity));
}

}  // namespace dtb
