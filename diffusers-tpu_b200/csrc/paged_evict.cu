// Eviction from a paged key/value cache by accumulated attention weight: a kernel that chooses the tokens of each head, and
// one that copies their rows to other pages.
//
// Choosing.  The k heaviest of n weights are those above the k-th largest, and of those equal to it as many as are
// missing, lowest slot first.  The k-th largest comes from three histograms of 11, 11 and 10 bits over the weights' bits,
// mapped so that unsigned order is weight order; a scan over the slots then gives each kept one its place.
// Copying.  Half a warp moves a row of 128 channels, 16 bytes a lane, with a few rows in flight.
#include <algorithm>

#include "host_common.h"
#include "paged.cuh"

namespace dtb {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kDigits = 2048;

// Unsigned order of the result is the order of the weights: -0 equals 0, NaN lies above infinity.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);          // -0 + 0 = 0
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive prefix sum over the block of one int a thread; every thread also gets the total.  Ends with a barrier.
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[31];
  const int before = (warp > 0 ? warp_sums[warp - 1] : 0) + incl - x;
  __syncthreads();
  return before;
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ dtb_paged_evict_params p) {
  __shared__ int hist[kDigits];
  __shared__ int warp_sums[32];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_left;
  const int b = blockIdx.y, h = blockIdx.x;
  const int len = table_len(p.kv_len, b, static_cast<int64_t>(p.table_width) * p.page_size);
  const int out_len = min(len, p.keep);
  int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.Hkv + h) * p.keep;
  const int out_cap = p.out_width * p.page_size;
  float* w_out = p.weights_out + (static_cast<int64_t>(b) * p.Hkv + h) * out_cap;
  const float* w = p.weights + b * p.w_stride_b + h * p.w_stride_h;
  if (h == 0 && threadIdx.x == 0) p.kv_len_out[b] = out_len;
  for (int i = out_len + threadIdx.x; i < p.keep; i += kSelectThreads) kept[i] = -1;
  for (int i = out_len + threadIdx.x; i < out_cap; i += kSelectThreads) w_out[i] = 0.f;
  if (len <= p.keep) {
    for (int i = threadIdx.x; i < len; i += kSelectThreads) {
      kept[i] = i;
      w_out[i] = w[i];
    }
    return;
  }
  const int old = len - p.recent;                        // slots to choose from
  const int k = p.keep - p.recent;
  uint32_t prefix = 0;                                   // leading bits of the k-th largest, in place
  int left = k;                                          // how many are still to be found among those with that prefix
  const int shifts[3] = {21, 10, 0};
  const int bits[3] = {11, 11, 10};
  if (k > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = threadIdx.x; i < kDigits; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      const int shift = shifts[pass], n = 1 << bits[pass];
      const uint32_t above = pass == 0 ? 0u : ~0u << (shift + bits[pass]);
      for (int i = threadIdx.x; i < old; i += kSelectThreads) {
        const uint32_t u = order_of(w[i]);
        if ((u & above) == prefix) atomicAdd(&hist[(u >> shift) & (n - 1)], 1);
      }
      __syncthreads();
      // digits from the top: the first at which the running count reaches `left` is the k-th largest's
      const int d0 = n - 1 - 2 * static_cast<int>(threadIdx.x);
      const int a0 = d0 >= 0 ? hist[d0] : 0, a1 = d0 >= 1 ? hist[d0 - 1] : 0;
      int total;
      const int before = block_scan(a0 + a1, warp_sums, total);
      if (before < left && before + a0 + a1 >= left) {
        const bool first = before + a0 >= left;
        sh_prefix = prefix | (static_cast<uint32_t>(first ? d0 : d0 - 1) << shift);
        sh_left = left - before - (first ? 0 : a0);
      }
      __syncthreads();
      prefix = sh_prefix;
      left = sh_left;
      __syncthreads();
    }
  }
  // `prefix` is the k-th largest and `left` the number of its equals that are kept
  int placed = 0, equals = 0;
  for (int base = 0; base < len; base += kSelectThreads) {
    const int i = base + threadIdx.x;
    float x = 0.f;
    bool over = false, same = false;
    if (i < len) {
      x = w[i];
      const uint32_t u = order_of(x);
      over = i >= old || (k > 0 && u > prefix);
      same = i < old && k > 0 && u == prefix;
    }
    int n_same, n_take;
    const int same_before = block_scan(same ? 1 : 0, warp_sums, n_same) + equals;
    const bool take = over || (same && same_before < left);
    const int at = block_scan(take ? 1 : 0, warp_sums, n_take) + placed;
    if (take) {
      kept[at] = i;
      w_out[at] = x;
    }
    equals += n_same;
    placed += n_take;
  }
}

constexpr int kCopyThreads = 256;
constexpr int kRowsInFlight = 4;

// Lanes of a row: D / 8, 16 bytes each.  A block copies rows of one head of one sequence.
__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const __grid_constant__ dtb_paged_evict_params p, int lanes, int rows_per_block) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int n = p.kv_len_out[b];
  const int first = blockIdx.x * rows_per_block;
  if (first >= n) return;
  const int last = min(first + rows_per_block, n);
  const int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.Hkv + h) * p.keep;
  const int32_t* from = p.page_table + b * p.table_stride;
  const int32_t* to = p.out_table + b * p.out_stride;
  const int step = kCopyThreads / lanes;
  const int lane = threadIdx.x % lanes, row = threadIdx.x / lanes;
  if (row >= step) return;
  char* kc = static_cast<char*>(p.key_cache);
  char* vc = static_cast<char*>(p.value_cache);
  for (int i0 = first + row; i0 < last; i0 += step * kRowsInFlight) {
    uint4 kx[kRowsInFlight], vx[kRowsInFlight];
    int page_out[kRowsInFlight];
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      const int i = i0 + u * step;
      page_out[u] = -1;
      kx[u] = vx[u] = make_uint4(0u, 0u, 0u, 0u);
      if (i >= last) continue;
      const int slot = kept[i];
      const int page = from[slot / p.page_size];
      page_out[u] = to[i / p.page_size];
      if (page < 0 || page >= p.pages) continue;
      const int64_t r = slot % p.page_size;
      kx[u] = reinterpret_cast<const uint4*>(kc + 2 * (page * p.kc_stride_p + h * p.kc_stride_h + r * p.kc_stride_r))[lane];
      vx[u] = reinterpret_cast<const uint4*>(vc + 2 * (page * p.vc_stride_p + h * p.vc_stride_h + r * p.vc_stride_r))[lane];
    }
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      if (page_out[u] < 0 || page_out[u] >= p.pages) continue;
      const int64_t r = (i0 + u * step) % p.page_size;
      const int64_t page = page_out[u];
      reinterpret_cast<uint4*>(kc + 2 * (page * p.kc_stride_p + h * p.kc_stride_h + r * p.kc_stride_r))[lane] = kx[u];
      reinterpret_cast<uint4*>(vc + 2 * (page * p.vc_stride_p + h * p.vc_stride_h + r * p.vc_stride_r))[lane] = vx[u];
    }
  }
}

}  // namespace
}  // namespace dtb

extern "C" int dtb_paged_evict(const dtb_paged_evict_params* ep, void* stream) {
  using namespace dtb;
  if (ep == nullptr || ep->key_cache == nullptr || ep->value_cache == nullptr || ep->weights == nullptr || ep->page_table == nullptr ||
      ep->out_table == nullptr || ep->kv_len == nullptr || ep->kept == nullptr || ep->weights_out == nullptr || ep->kv_len_out == nullptr)
    return DTB_ERR_NULL;
  if (ep->B < 0 || ep->Hkv <= 0 || ep->pages < 0 || ep->page_size <= 0 || ep->table_width < 0 || ep->out_width <= 0) return DTB_ERR_SHAPE;
  if (ep->D <= 0 || ep->D % 8 != 0 || ep->D / 8 > kCopyThreads) return DTB_ERR_SHAPE;
  const int64_t out_cap = static_cast<int64_t>(ep->out_width) * ep->page_size;
  if (static_cast<int64_t>(ep->table_width) * ep->page_size > 0x7fffffff - kSelectThreads || out_cap > 0x7fffffff - kSelectThreads) return DTB_ERR_SHAPE;
  if (ep->keep < 1 || ep->keep > out_cap || ep->recent < 0 || ep->recent > ep->keep) return DTB_ERR_SHAPE;
  if (ep->Hkv > 65535 || ep->B > 65535) return DTB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(ep->key_cache) & 15u) || (reinterpret_cast<uintptr_t>(ep->value_cache) & 15u)) return DTB_ERR_ALIGN;
  for (int64_t st : {ep->kc_stride_p, ep->kc_stride_h, ep->kc_stride_r, ep->vc_stride_p, ep->vc_stride_h, ep->vc_stride_r})
    if (st % 8 != 0) return DTB_ERR_ALIGN;
  if (ep->B == 0) return DTB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  evict_select_kernel<<<dim3(ep->Hkv, ep->B), kSelectThreads, 0, s>>>(*ep);
  if (!launch_ok("evict_select_kernel launch")) return DTB_ERR_LAUNCH;
  const int lanes = ep->D / 8;
  const int rows = (kCopyThreads / lanes) * kRowsInFlight;
  const unsigned blocks = static_cast<unsigned>((ep->keep + rows - 1) / rows);
  evict_copy_kernel<<<dim3(blocks, ep->Hkv, ep->B), kCopyThreads, 0, s>>>(*ep, lanes, rows);
  return launch_ok("evict_copy_kernel launch") ? DTB_OK : DTB_ERR_LAUNCH;
}
