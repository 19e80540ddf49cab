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

// Slot of the first of a sequence's n new tokens: where paged_append puts it.  A length past the table keeps the new tokens' slots
// as long as the first of them has one; where none has, they count as the last ones of the table.
__device__ __forceinline__ int first_slot(const int32_t* kv_len, int b, int n, int64_t capacity) {
  const int64_t at = static_cast<int64_t>(max(__ldg(kv_len + b), 0)) - n;
  return static_cast<int>(at < capacity ? at : capacity - n);
}

}  // namespace dtb
