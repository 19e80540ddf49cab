// Attention of new tokens over a paged key/value cache, and the attention that each key got.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "host_common.h"
#include "paged_attn.cuh"
#include "paged_weights.cuh"

namespace dtb {
namespace {

constexpr float kLog2e = 1.44269504f;

int check_cache(const void* cache, int64_t sp, int64_t sh, int64_t sr, int pages, int Hkv, int page_size) {
  if ((reinterpret_cast<uintptr_t>(cache) & 15u) || sp % 8 || sh % 8 || sr % 8) return DTB_ERR_ALIGN;
  // an axis of more than one entry needs a positive stride (tensor-map rule)
  if ((pages > 1 && sp <= 0) || (Hkv > 1 && sh <= 0) || (page_size > 1 && sr <= 0)) return DTB_ERR_SHAPE;
  return DTB_OK;
}

template <class P>
int check_batch(const P* p) {
  if (p->dtype != DTB_BF16 && p->dtype != DTB_FP16) return DTB_ERR_DTYPE;
  if (p->D != 64 && p->D != 128) return DTB_ERR_SHAPE;
  if (p->B < 0 || p->T < 0 || p->Hkv <= 0 || p->Hq <= 0 || p->Hq % p->Hkv != 0 || p->Hq / p->Hkv > 128) return DTB_ERR_SHAPE;
  if (p->pages < 0 || p->table_width < 0 || p->window < 0 || (p->window > 0 && !p->causal)) return DTB_ERR_SHAPE;
  const int ps = p->page_size;
  if (!(ps == 8 || ps == 16 || ps == 32 || ps == 64 || (ps > 0 && ps % 128 == 0))) return DTB_ERR_SHAPE;
  if (static_cast<int64_t>(p->table_width) * ps > 0x7ffffc00) return DTB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(p->q) & 15u) || p->q_stride_t % 8 || p->q_stride_h % 8) return DTB_ERR_ALIGN;
  if ((p->T > 1 && p->q_stride_t <= 0) || (p->Hq > 1 && p->q_stride_h <= 0)) return DTB_ERR_SHAPE;
  return check_cache(p->key_cache, p->kc_stride_p, p->kc_stride_h, p->kc_stride_r, p->pages, p->Hkv, ps);
}

}  // namespace
}  // namespace dtb

namespace dtb {
namespace {

// What a key tile costs, in eighths of one of a unit that waits for memory: in the kernel of few rows, whose other units lack
// registers, with one query tile and two, and with two in the other kernel.  47 single tokens x 24 heads over 2000-32768 keys
// beside a chunk of 64 tokens: 606 us with all tiles alike (12 for two query tiles), 496 with 16, 383 with 24, 371 with 32 (40
// heads: 573, 489, 388, 396); beside a chunk of 512: 541 us with all alike, 495 with 11, 511 with 14.
constexpr int kThinCostOne = 12, kThinCostTwo = 24, kCostTwo = 11;

// Blocks of a launch: one a SM.  The plan divides any amount of work among them.
int plan_blocks() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && sms > 0)
    return std::min(sms, kPlanMaxBlocks);
  (void)cudaGetLastError();
  return 148;
}

// 4-D map of 16-bit elements with a contiguous first axis, boxes of 64 channels in the 128-byte swizzle.
int encode_map(CUtensorMap* out, const void* base, bool bf16, const int64_t (&dims)[4], const int64_t (&strides)[3], const int (&box)[3]) {
  EncodeTiledFn enc = get_encode_tiled();
  if (enc == nullptr) {
    set_detail("cuTensorMapEncodeTiled entry point not found");
    return DTB_ERR_LAUNCH;
  }
  cuuint64_t d[4], st[3];
  for (int i = 0; i < 4; ++i) d[i] = static_cast<cuuint64_t>(dims[i]);
  // an axis of one entry may come with any stride; give it a harmless legal one
  for (int i = 0; i < 3; ++i) st[i] = dims[i + 1] > 1 ? static_cast<cuuint64_t>(strides[i] * 2) : 256;
  const cuuint32_t b[4] = {64, static_cast<cuuint32_t>(box[0]), static_cast<cuuint32_t>(box[1]), static_cast<cuuint32_t>(box[2])};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(out, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), d, st, b, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return DTB_OK;
  set_detail("cuTensorMapEncodeTiled failed for a paged call");
  return DTB_ERR_LAUNCH;
}

int encode_cache(CUtensorMap* out, const void* cache, bool bf16, int D, int page_size, int Hkv, int pages, int64_t sp, int64_t sh, int64_t sr) {
  return encode_map(out, cache, bf16, {D, page_size, Hkv, std::max(pages, 1)}, {sr, sh, sp}, {std::min(page_size, kBlockN), 1, 1});
}

// New tokens as [key head, token, head of the group, channel]: a box is a tile's tokens with all heads of the group.
int encode_queries(CUtensorMap* out, const void* q, bool bf16, int D, int Hkv, int G, int T, int tile_tokens, int64_t st, int64_t sh) {
  return encode_map(out, q, bf16, {D, G, T, Hkv}, {sh, st, sh * G}, {G, tile_tokens, 1});
}

// Whether a unit of so many slots may be cut: not without kLeastKeys on both sides.
bool may_cut(int64_t capacity) { return capacity >= 2 * kLeastKeys; }

template <class E, int kD, bool kThin>
int launch_paged(const PagedKernelParams& kp, int blocks, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (!cuda_ok(cudaGetDevice(&dev), "cudaGetDevice")) return DTB_ERR_LAUNCH;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    const void* fn = reinterpret_cast<const void*>(paged_attn_kernel<E, kD, kThin>);
    cudaFuncAttributes fa;
    if (!cuda_ok(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kPagedSmem<kD>)), "cudaFuncSetAttribute") ||
        !cuda_ok(cudaFuncGetAttributes(&fa, fn), "cudaFuncGetAttributes"))
      return DTB_ERR_LAUNCH;
    if (fa.numRegs != kLaunchRegs) {
      set_detail("paged_attn_kernel was not compiled for the registers that its warpgroups hand over");
      return DTB_ERR_LAUNCH;
    }
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  paged_attn_kernel<E, kD, kThin><<<blocks, kPagedThreads, kPagedSmem<kD>, s>>>(kp);
  if (!launch_ok("paged_attn_kernel launch")) return DTB_ERR_LAUNCH;
  if (!may_cut(kp.plan.capacity)) return DTB_OK;
  // The merge's blocks are set up while the attention kernel runs; they wait for its end themselves.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, kThin ? 4 : 16);              // units of 16 rows mostly, and of up to 256
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_ok(cudaLaunchKernelEx(&cfg, paged_merge_kernel<E, kD>, static_cast<const float*>(kp.slots), static_cast<const MergeDesc*>(kp.merge),
                                    static_cast<E*>(kp.o), kp.o_stride_t, kp.o_stride_h, kp.lse, kp.Hq, kp.G, kp.tile_tokens),
                 "paged_merge_kernel launch") ? DTB_OK : DTB_ERR_LAUNCH;
}

template <class E, int kD>
int launch_weights(const WeightsKernelParams& kp, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (!cuda_ok(cudaGetDevice(&dev), "cudaGetDevice")) return DTB_ERR_LAUNCH;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    if (!cuda_ok(cudaFuncSetAttribute(reinterpret_cast<const void*>(key_weights_kernel<E, kD>), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(kWeightsSmem<kD>)), "cudaFuncSetAttribute"))
      return DTB_ERR_LAUNCH;
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  key_weights_kernel<E, kD><<<plan_blocks(), kWeightsThreads, kWeightsSmem<kD>, s>>>(kp);
  return launch_ok("key_weights_kernel launch") ? DTB_OK : DTB_ERR_LAUNCH;
}

// States of the pieces, where there may be any.
size_t slot_bytes(const dtb_paged_attn_params* p, int blocks) {
  return may_cut(static_cast<int64_t>(p->table_width) * p->page_size) ? static_cast<size_t>(2) * blocks * kSlotRows * (p->D + 2) * sizeof(float) : 0;
}

}  // namespace
}  // namespace dtb

extern "C" size_t dtb_paged_attn_workspace_bytes(const dtb_paged_attn_params* p) {
  using namespace dtb;
  if (p == nullptr || p->B <= 0 || p->T <= 0 || p->D <= 0) return 0;
  const int blocks = plan_blocks();
  return slot_bytes(p, blocks) + blocks * sizeof(MergeDesc);
}

extern "C" int dtb_paged_attn(const dtb_paged_attn_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dtb;
  if (p == nullptr) return DTB_ERR_NULL;
  if (p->B == 0 || p->T == 0) return check_batch(p);
  if (p->q == nullptr || p->key_cache == nullptr || p->value_cache == nullptr || p->o == nullptr || p->page_table == nullptr ||
      p->query_start == nullptr || p->kv_len == nullptr)
    return DTB_ERR_NULL;
  if (const int st = check_batch(p)) return st;
  if (const int st = check_cache(p->value_cache, p->vc_stride_p, p->vc_stride_h, p->vc_stride_r, p->pages, p->Hkv, p->page_size)) return st;
  if ((reinterpret_cast<uintptr_t>(p->o) & 15u) || p->o_stride_t % 8 || p->o_stride_h % 8) return DTB_ERR_ALIGN;
  if (p->B > kPlanMaxSeqs) return DTB_ERR_SHAPE;
  if (!device_is_sm100()) return DTB_ERR_ARCH;
  const int blocks = plan_blocks();
  if (workspace == nullptr || workspace_bytes < dtb_paged_attn_workspace_bytes(p)) return DTB_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15u) return DTB_ERR_ALIGN;
  const bool bf16 = p->dtype == DTB_BF16;
  PagedKernelParams kp;
  kp.G = p->Hq / p->Hkv;
  kp.tile_tokens = kBlockM / kp.G;
  // with no page to read every copy lies past the end of the map, whose memory has to exist all the same
  const void* kc = p->pages > 0 ? p->key_cache : p->q;
  const void* vc = p->pages > 0 ? p->value_cache : p->q;
  int st = encode_queries(&kp.tmap_q, p->q, bf16, p->D, p->Hkv, kp.G, p->T, kp.tile_tokens, p->q_stride_t, p->q_stride_h);
  if (st == DTB_OK) st = encode_cache(&kp.tmap_k, kc, bf16, p->D, p->page_size, p->Hkv, p->pages, p->kc_stride_p, p->kc_stride_h, p->kc_stride_r);
  if (st == DTB_OK) st = encode_cache(&kp.tmap_v, vc, bf16, p->D, p->page_size, p->Hkv, p->pages, p->vc_stride_p, p->vc_stride_h, p->vc_stride_r);
  if (st != DTB_OK) return st;
  kp.plan = {p->query_start, p->kv_len, static_cast<int64_t>(p->table_width) * p->page_size, p->B, p->T, p->Hkv, 2 * kp.tile_tokens, p->causal, p->window};
  kp.page_table = p->page_table;
  kp.table_stride = p->table_stride;
  kp.table_width = p->table_width;
  kp.pages = p->pages;
  kp.page_size = p->page_size;
  kp.o = p->o;
  kp.o_stride_t = p->o_stride_t;
  kp.o_stride_h = p->o_stride_h;
  kp.lse = p->lse;
  kp.slots = static_cast<float*>(workspace);
  kp.merge = reinterpret_cast<MergeDesc*>(static_cast<char*>(workspace) + slot_bytes(p, blocks));
  kp.status = p->status;
  kp.Hq = p->Hq;
  kp.scale_log2 = (p->scale > 0.f ? p->scale : 1.0f / sqrtf(static_cast<float>(p->D))) * kLog2e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Whether units have few rows, the device knows; the host, how many they have in the mean.
  kp.plan.tile_tokens = kp.tile_tokens;
  if (static_cast<int64_t>(p->T) * kp.G <= static_cast<int64_t>(p->B) * kThinRows) {
    // beside units of few rows, which wait for memory, a key tile of others takes half as long again, or twice as long
    kp.plan.cheap_tokens = kThinRows / kp.G;
    kp.plan.cost_one = kThinCostOne;
    kp.plan.cost_two = kThinCostTwo;
    if (p->D == 128) return bf16 ? launch_paged<__nv_bfloat16, 128, true>(kp, blocks, s) : launch_paged<__half, 128, true>(kp, blocks, s);
    return bf16 ? launch_paged<__nv_bfloat16, 64, true>(kp, blocks, s) : launch_paged<__half, 64, true>(kp, blocks, s);
  }
  kp.plan.cheap_tokens = kp.tile_tokens;
  kp.plan.cost_two = kCostTwo;
  if (p->D == 128) return bf16 ? launch_paged<__nv_bfloat16, 128, false>(kp, blocks, s) : launch_paged<__half, 128, false>(kp, blocks, s);
  return bf16 ? launch_paged<__nv_bfloat16, 64, false>(kp, blocks, s) : launch_paged<__half, 64, false>(kp, blocks, s);
}

extern "C" int dtb_paged_key_weights(const dtb_paged_key_weights_params* p, void* stream) {
  using namespace dtb;
  if (p == nullptr) return DTB_ERR_NULL;
  if (p->B == 0 || p->table_width == 0) return check_batch(p);
  if (p->key_cache == nullptr || p->out == nullptr || p->page_table == nullptr || p->query_start == nullptr || p->kv_len == nullptr)
    return DTB_ERR_NULL;
  if (p->T > 0 && (p->q == nullptr || p->lse == nullptr)) return DTB_ERR_NULL;    // without new tokens there are none to read
  if (const int st = check_batch(p)) return st;
  if (p->B > kPlanMaxSeqs) return DTB_ERR_SHAPE;
  if (!device_is_sm100()) return DTB_ERR_ARCH;
  const bool bf16 = p->dtype == DTB_BF16;
  WeightsKernelParams kp;
  kp.G = p->Hq / p->Hkv;
  const int tile_tokens = kBlockM / kp.G;
  // as in dtb_paged_attn; without new tokens there are no queries to map either
  const void* any = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(p->out) & ~static_cast<uintptr_t>(15));
  const void* q = p->T > 0 ? p->q : any;
  const void* kc = p->pages > 0 ? p->key_cache : any;
  int st = encode_queries(&kp.tmap_q, q, bf16, p->D, p->Hkv, kp.G, std::max(p->T, 1), tile_tokens, p->q_stride_t, p->q_stride_h);
  if (st == DTB_OK) st = encode_cache(&kp.tmap_k, kc, bf16, p->D, p->page_size, p->Hkv, p->pages, p->kc_stride_p, p->kc_stride_h, p->kc_stride_r);
  if (st != DTB_OK) return st;
  kp.plan = {p->query_start, p->kv_len, static_cast<int64_t>(p->table_width) * p->page_size, p->B, p->T, p->Hkv, tile_tokens, p->causal, p->window};
  kp.page_table = p->page_table;
  kp.table_stride = p->table_stride;
  kp.pages = p->pages;
  kp.page_size = p->page_size;
  kp.lse = p->lse;
  kp.prior = p->prior;
  kp.out = p->out;
  kp.prior_stride_b = p->prior_stride_b;
  kp.prior_stride_h = p->prior_stride_h;
  kp.out_stride_b = p->out_stride_b;
  kp.out_stride_h = p->out_stride_h;
  kp.status = p->status;
  kp.Hq = p->Hq;
  kp.scale_log2 = (p->scale > 0.f ? p->scale : 1.0f / sqrtf(static_cast<float>(p->D))) * kLog2e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->D == 128) return bf16 ? launch_weights<__nv_bfloat16, 128>(kp, s) : launch_weights<__half, 128>(kp, s);
  return bf16 ? launch_weights<__nv_bfloat16, 64>(kp, s) : launch_weights<__half, 64>(kp, s);
}
