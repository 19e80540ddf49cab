// Stand-ins for what the plan of the paged kernels uses of CUDA: a block's threads are host threads that meet at barriers.
#pragma once
#include <algorithm>
#include <atomic>
#include <barrier>
#include <cstdint>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
#define __global__
using std::max;
using std::min;
struct int2 { int x, y; };
struct int3 { int x, y, z; };
inline int2 make_int2(int x, int y) { return {x, y}; }
inline int3 make_int3(int x, int y, int z) { return {x, y, z}; }
template <class T> inline T __ldg(const T* p) { return *p; }
struct Dim { int x; };
inline thread_local Dim threadIdx;
inline std::barrier<>* block_barrier;
inline std::vector<std::barrier<>*> warp_barriers;
inline int64_t lanes_of[1024];
inline std::atomic<int> any_of{0};
inline void __syncthreads() { block_barrier->arrive_and_wait(); }
inline int __syncthreads_or(int x) {
  __syncthreads();
  any_of = 0;
  __syncthreads();
  if (x) any_of = 1;
  __syncthreads();
  return any_of;
}
template <class T> inline T __shfl_up_sync(unsigned, T x, int o) {
  const int t = threadIdx.x, warp = t / 32;
  lanes_of[t] = static_cast<int64_t>(x);
  warp_barriers[warp]->arrive_and_wait();
  const T y = static_cast<T>((t & 31) >= o ? lanes_of[t - o] : lanes_of[t]);
  warp_barriers[warp]->arrive_and_wait();
  return y;
}
