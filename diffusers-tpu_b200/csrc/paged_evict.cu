// Eviction from a paged key/value cache by accumulated attention weight: a kernel that chooses the tokens of each head, and
// one that copies their rows to other pages.
//
// Choosing.  The k heaviest of n weights are those above the k-th largest, and of those equal to it as many as are
// missing, lowest slot first.  The k-th largest comes from three histograms of 11, 11 and 10 bits over the weights' bits,
// mapped so that unsigned order is weight order.  A head is a cluster of up to eight blocks whose warps have a run of slots each;
// histograms, and how many each warp keeps, are added up through the cluster's shared memory, and a warp that knows how many
// stay before its run writes its own.  (A block a head that scanned 1024 slots at a time took 89 us for 32 heads of 50000-65536
// slots, most of it at barriers.)
// Copying.  Bound by bytes: each kept row read once and written once.  D / 8 lanes move a row, 16 bytes each, four rows of both
// caches in flight, with the places of the next four looked up under them.
#include <algorithm>

#include "host_common.h"
#include "paged.cuh"

namespace dtb {
namespace {

constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32;
constexpr int kDigits = 2048;

// Unsigned order of the result is the order of the weights: -0 equals 0, NaN lies above infinity.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);          // -0 + 0 = 0
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int kMostBlocks = 8;             // of a head
constexpr int kBatch = 8;                  // weights of a lane asked for at a time
// Slots of a sequence: places are ints, and rounded up to 32 for each of a cluster's 128 warps, or to a copy's block of up to 4096 rows.
constexpr int kMostSlots = 0x7fffffff - 8192;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync(int blocks) {
  if (blocks == 1) {
    __syncthreads();
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// An int of another block's shared memory, at the address that it has in this one's.
__device__ __forceinline__ int peer_int(const int* mine, uint32_t rank) {
  uint32_t a;
  int x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
  return x;
}

// Inclusive sum over the lanes of a warp.
__device__ __forceinline__ int warp_scan(int x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// `blocks` is the size of the cluster, blockIdx.x the head times it.
__global__ void __launch_bounds__(kSelectThreads, 2) evict_select_kernel(const __grid_constant__ dtb_paged_evict_params p, int blocks) {
  __shared__ int hist[2][kDigits];                       // the passes' in turn: one is read by the cluster, the next one cleared
  __shared__ int groups[2][kDigits / 32];
  __shared__ int counts[2 * 32];                            // this block's warps: kept whatever, and equal to the k-th largest
  __shared__ int before[2 * 32];                         // of this block's warps: what the warps before them have of both
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_left;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_rank());
  const int b = blockIdx.y, h = blockIdx.x / blocks;
  const int len = table_len(p.kv_len, b, static_cast<int64_t>(p.table_width) * p.page_size);
  const int out_len = min(len, p.keep);
  int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.Hkv + h) * p.keep;
  const int out_cap = p.out_width * p.page_size;
  float* w_out = p.weights_out + (static_cast<int64_t>(b) * p.Hkv + h) * out_cap;
  const float* w = p.weights + b * p.w_stride_b + h * p.w_stride_h;
  const int step = blocks * kSelectThreads;
  if (h == 0 && rank == 0 && tid == 0) p.kv_len_out[b] = out_len;
  for (int i = out_len + rank * kSelectThreads + tid; i < p.keep; i += step) kept[i] = -1;
  for (int i = out_len + rank * kSelectThreads + tid; i < out_cap; i += step) w_out[i] = 0.f;
  if (len <= p.keep) {                                   // the same for all blocks of the cluster
    for (int i = rank * kSelectThreads + tid; i < len; i += step) {
      kept[i] = i;
      w_out[i] = w[i];
    }
    return;
  }
  const int old = len - p.recent;                        // slots to choose from
  const int k = p.keep - p.recent;
  // this warp's run of slots
  const int warps = blocks * kSelectWarps;
  const int run = ((len + warps - 1) / warps + 31) & ~31;
  const int run0 = min((rank * kSelectWarps + warp) * run, len), run1 = min(run0 + run, len);
  // f(slot, weight) for each slot of the run below `end`, a warp's 32 neighbours at a time; slots past the end come with `in` false
  auto over_run = [&](int end, auto f) {
    for (int i0 = run0; i0 < end; i0 += 32 * kBatch) {
      float x[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * 32 + lane;
        x[u] = i < end ? w[i] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i0 + u * 32 < end) f(i0 + u * 32 + lane, x[u], i0 + u * 32 + lane < end);
    }
  };
  uint32_t prefix = 0;                                   // leading bits of the k-th largest, in place
  int left = k;                                          // how many are still to be found among those with that prefix
  // sum over the cluster's first blocks of the int at `mine` of each one's shared memory
  auto cluster_sum = [&](const int* mine, int ranks) {
    int v[kMostBlocks], sum = 0;
#pragma unroll
    for (int r = 0; r < kMostBlocks; ++r)
      if (r < ranks) v[r] = peer_int(mine, r);
#pragma unroll
    for (int r = 0; r < kMostBlocks; ++r)
      if (r < ranks) sum += v[r];
    return sum;
  };
  if (k > 0) {
    for (int i = tid; i < kDigits; i += kSelectThreads) hist[0][i] = 0;
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, n = 1 << bits;
      int* count = hist[pass & 1];
      const uint32_t above = pass == 0 ? 0u : ~0u << (shift + bits);
      over_run(min(run1, old), [&](int, float x, bool in) {
        const uint32_t u = order_of(x);
        if (in && (u & above) == prefix) atomicAdd(&count[(u >> shift) & (n - 1)], 1);
      });
      __syncthreads();
      for (int g = warp; g < n / 32; g += kSelectWarps) {  // sums of 32 digits each
        const int sum = __reduce_add_sync(0xffffffffu, count[g * 32 + lane]);
        if (lane == 0) groups[pass & 1][g] = sum;
      }
      cluster_sync(blocks);
      for (int i = tid; i < kDigits; i += kSelectThreads) hist[~pass & 1][i] = 0;
      // From the top, the first group and then the first digit of it at which the running count reaches `left`: the k-th
      // largest's.  (Sums of all 2048 digits through the cluster, 32 remote loads a thread: 84 us a choice of 32 heads.)
      if (warp == 0) {
        int seen = 0, at = 0;
        for (int g0 = n / 32 - 1; g0 >= 0; g0 -= 32) {
          const int mine = cluster_sum(&groups[pass & 1][g0 - lane], blocks);
          const int inc = seen + warp_scan(mine);
          const uint32_t reached = __ballot_sync(0xffffffffu, inc >= left);
          if (reached) {
            const int first = __ffs(reached) - 1;
            at = g0 - first;
            seen = __shfl_sync(0xffffffffu, inc - mine, first);
            break;
          }
          seen = __shfl_sync(0xffffffffu, inc, 31);
        }
        const int mine = cluster_sum(&count[at * 32 + 31 - lane], blocks);
        const int inc = seen + warp_scan(mine);
        const uint32_t reached = __ballot_sync(0xffffffffu, inc >= left);
        const int first = __ffs(reached) - 1;
        if (lane == first) {
          sh_prefix = prefix | (static_cast<uint32_t>(at * 32 + 31 - lane) << shift);
          sh_left = left - (inc - mine);
        }
      }
      __syncthreads();
      prefix = sh_prefix;
      left = sh_left;
    }
  }
  // `prefix` is the k-th largest and `left` the number of its equals that stay
  auto stays = [&](int i, float x) { return i >= old || (k > 0 && order_of(x) > prefix); };
  auto equals = [&](int i, float x) { return i < old && k > 0 && order_of(x) == prefix; };
  int n_stay = 0, n_equal = 0;
  over_run(run1, [&](int i, float x, bool in) {
    n_stay += __popc(__ballot_sync(0xffffffffu, in && stays(i, x)));
    n_equal += __popc(__ballot_sync(0xffffffffu, in && equals(i, x)));
  });
  if (lane == 0) {
    counts[warp] = n_stay;
    counts[32 + warp] = n_equal;
  }
  cluster_sync(blocks);
  // sums over the blocks before this one, and over this one's warps before each
  if (warp < 2) {
    const bool has = lane < kSelectWarps;
    const int sum = has ? cluster_sum(&counts[warp * 32 + lane], rank) : 0;
    const int all = __shfl_sync(0xffffffffu, warp_scan(sum), 31);
    const int mine = has ? counts[warp * 32 + lane] : 0;
    before[warp * 32 + lane] = all + warp_scan(mine) - mine;
  }
  cluster_sync(blocks);                                        // no block leaves while another reads its counts
  int stay_before = before[warp], equal_before = before[32 + warp];
  over_run(run1, [&](int i, float x, bool in) {
    const bool s = in && stays(i, x), e = in && equals(i, x);
    const uint32_t s_votes = __ballot_sync(0xffffffffu, s), e_votes = __ballot_sync(0xffffffffu, e), lower = (1u << lane) - 1;
    const int e_at = equal_before + __popc(e_votes & lower), s_at = stay_before + __popc(s_votes & lower);
    if (s || (e && e_at < left)) {
      const int at = s_at + min(e_at, left);             // equals before it that stay
      kept[at] = i;
      w_out[at] = x;
    }
    stay_before += __popc(s_votes);
    equal_before += __popc(e_votes);
  });
}

constexpr int kCopyThreads = 256;
constexpr int kRowsInFlight = 4;

// Lanes of a row: D / 8, 16 bytes each.  A block copies `rounds` x step x kRowsInFlight rows of one head of one sequence.
__global__ void __launch_bounds__(kCopyThreads, 4) evict_copy_kernel(const __grid_constant__ dtb_paged_evict_params p, int lanes, int rounds, int page_shift) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.z, h = blockIdx.y;
  const int n = p.kv_len_out[b];
  const int step = kCopyThreads / lanes;
  const int first = blockIdx.x * rounds * step * kRowsInFlight;
  if (first >= n) return;
  const int last = min(first + rounds * step * kRowsInFlight, n);
  const int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.Hkv + h) * p.keep;
  const int32_t* from = p.page_table + b * p.table_stride;
  const int32_t* to = p.out_table + b * p.out_stride;
  const int lane = threadIdx.x % lanes, row = threadIdx.x / lanes;
  if (row >= step) return;
  char* kc = static_cast<char*>(p.key_cache) + 2 * (h * p.kc_stride_h) + lane * 16;
  char* vc = static_cast<char*>(p.value_cache) + 2 * (h * p.vc_stride_h) + lane * 16;
  auto page_number = [&](int i) { return page_shift >= 0 ? i >> page_shift : i / p.page_size; };
  int page_in[kRowsInFlight], row_in[kRowsInFlight], page_out[kRowsInFlight];
  auto look_up = [&](int i0) {
    int slot[kRowsInFlight];
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) slot[u] = i0 + u * step < last ? kept[i0 + u * step] : -1;
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      page_in[u] = page_out[u] = -1;
      row_in[u] = 0;
      if (slot[u] < 0) continue;
      const int q = page_number(slot[u]);
      row_in[u] = slot[u] - q * p.page_size;
      page_in[u] = from[q];
      page_out[u] = to[page_number(i0 + u * step)];
    }
  };
  look_up(first + row);
  for (int i0 = first + row; i0 < last; i0 += step * kRowsInFlight) {
    uint4 kx[kRowsInFlight], vx[kRowsInFlight];
    int64_t k_to[kRowsInFlight], v_to[kRowsInFlight];
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      kx[u] = vx[u] = make_uint4(0u, 0u, 0u, 0u);
      const int64_t page = page_in[u];
      if (page >= 0 && page < p.pages) {
        kx[u] = *reinterpret_cast<const uint4*>(kc + 2 * (page * p.kc_stride_p + row_in[u] * p.kc_stride_r));
        vx[u] = *reinterpret_cast<const uint4*>(vc + 2 * (page * p.vc_stride_p + row_in[u] * p.vc_stride_r));
      }
      const int64_t out = page_out[u];
      const int i = i0 + u * step, r = i - page_number(i) * p.page_size;
      k_to[u] = out >= 0 && out < p.pages ? 2 * (out * p.kc_stride_p + r * p.kc_stride_r) : -1;
      v_to[u] = 2 * (out * p.vc_stride_p + r * p.vc_stride_r);
    }
    look_up(i0 + step * kRowsInFlight);
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      if (k_to[u] < 0) continue;
      *reinterpret_cast<uint4*>(kc + k_to[u]) = kx[u];
      *reinterpret_cast<uint4*>(vc + v_to[u]) = vx[u];
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
  if (static_cast<int64_t>(ep->table_width) * ep->page_size > kMostSlots || out_cap > kMostSlots) return DTB_ERR_SHAPE;
  if (ep->keep < 1 || ep->keep > out_cap || ep->recent < 0 || ep->recent > ep->keep) return DTB_ERR_SHAPE;
  if (ep->Hkv > 65535 || ep->B > 65535) return DTB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(ep->key_cache) & 15u) || (reinterpret_cast<uintptr_t>(ep->value_cache) & 15u)) return DTB_ERR_ALIGN;
  for (int64_t st : {ep->kc_stride_p, ep->kc_stride_h, ep->kc_stride_r, ep->vc_stride_p, ep->vc_stride_h, ep->vc_stride_r})
    if (st % 8 != 0) return DTB_ERR_ALIGN;
  if (ep->B == 0) return DTB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // A head's cluster: two blocks' worth of slots a block at least, and no more blocks than the chip holds at once.
  const int64_t capacity = static_cast<int64_t>(ep->table_width) * ep->page_size, heads = static_cast<int64_t>(ep->B) * ep->Hkv;
  int blocks = 1;
  while (blocks < kMostBlocks && capacity >= 4 * blocks * kSelectThreads && heads * blocks * 2 <= 296) blocks *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ep->Hkv * blocks, ep->B);
  cfg.blockDim = dim3(kSelectThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!cuda_ok(cudaLaunchKernelEx(&cfg, evict_select_kernel, *ep, blocks), "evict_select_kernel launch")) return DTB_ERR_LAUNCH;
  // The copies' blocks are set up while the choice is made; they wait for its end themselves.
  const int lanes = ep->D / 8;
  const int rows = (kCopyThreads / lanes) * kRowsInFlight;
  // a few rounds a block where there are rows enough for every SM to have several blocks all the same
  const int rounds = static_cast<int>(std::max<int64_t>(std::min<int64_t>(4, heads * ep->keep / (static_cast<int64_t>(rows) * 148 * 16)), 1));
  int page_shift = -1;                                   // of page sizes that are powers of two
  if ((ep->page_size & (ep->page_size - 1)) == 0)
    do ++page_shift; while (1 << page_shift < ep->page_size);
  cfg.gridDim = dim3((ep->keep + rows * rounds - 1) / (rows * rounds), ep->Hkv, ep->B);
  cfg.blockDim = dim3(kCopyThreads);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  return cuda_ok(cudaLaunchKernelEx(&cfg, evict_copy_kernel, *ep, lanes, rounds, page_shift), "evict_copy_kernel launch") ? DTB_OK : DTB_ERR_LAUNCH;
}
