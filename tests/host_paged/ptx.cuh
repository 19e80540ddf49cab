// Host stand-ins for what the paged attention kernel uses beside the other attention kernels' (host_trace/ptx.cuh, copied here as
// trace_ptx.cuh): one thread at a time, printing what it does.
#pragma once

#include <atomic>
#include <functional>
#include <type_traits>
#include <vector>

#define mbar_wait recorded_wait
#include "trace_ptx.cuh"
#undef mbar_wait
#define __noinline__

struct int2 { int x, y; };
struct int3 { int x, y, z; };
struct uint2 { unsigned x, y; };
inline int2 make_int2(int x, int y) { return {x, y}; }
inline int3 make_int3(int x, int y, int z) { return {x, y, z}; }
inline uint2 make_uint2(unsigned x, unsigned y) { return {x, y}; }
struct __half { uint16_t bits; };
extern Index3 gridDim;

namespace dtb {

template <class T> T __ldg(const T* p) { return *p; }
template <class T> T __shfl_up_sync(uint32_t, T x, int) { return x; }
template <class T> T __shfl_xor_sync(uint32_t, T x, int) { return x; }
template <class T> T __shfl_sync(uint32_t, T x, int) { return x; }
inline uint32_t __ballot_sync(uint32_t, bool x) { return x; }
inline int __syncthreads_or(int x) { __syncthreads(); return x; }

// A thread that waits for the description of a unit finds it in its place, as if the warp that describes it had come by.
inline std::function<void(uint32_t)> describe;
inline bool mbar_wait(uint32_t bar, uint32_t parity, const AbortCtx& ctx, int site) {
  if (describe) describe(bar);
  return recorded_wait(bar, parity, ctx, site);
}
inline void tmem_ld16_sync(uint32_t col, uint32_t* r) {
  record("ld %u 16\n", col & 0xffff);
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(growing ? 100.f * static_cast<float>(tiles_read) : 0.f);
  tiles_read += (col & 0xffff) == 0;
}

}  // namespace dtb
