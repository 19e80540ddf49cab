// Attention of new tokens over a paged key/value cache, and the attention that each key got.
#include <cmath>

#include "host_common.h"
#include "paged.cuh"

namespace dtb {
namespace {

constexpr float kLog2e = 1.44269504f;

__device__ __forceinline__ float value_at(const void* p, int64_t i, int dtype) {
  return dtype == DTB_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void put(void* p, int64_t i, int dtype, float x) {
  if (dtype == DTB_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// Keys [lo, hi) that new token i of n sees in a sequence of `len`.
__device__ __forceinline__ int2 seen(int len, int n, int i, int causal, int window) {
  if (!causal) return make_int2(0, len);
  const int hi = len - n + i + 1;
  return make_int2(window > 0 ? max(hi - window, 0) : 0, max(hi, 0));
}

// A warp per (token, query head); keys one after the other, a lane holds D / 32 channels.
__global__ void __launch_bounds__(128) paged_rows_kernel(const __grid_constant__ dtb_paged_attn_params p, float scale_log2) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<int64_t>(p.T) * p.Hq) return;
  const int t = static_cast<int>(row / p.Hq), h = static_cast<int>(row % p.Hq), hk = h / (p.Hq / p.Hkv);
  const int b = sequence_of(p.query_start, p.B, t);
  if (b < 0) return;
  const int2 rows = new_rows(p.query_start, b, p.T);
  const int len = table_len(p.kv_len, b, static_cast<int64_t>(p.table_width) * p.page_size);
  const int2 keys = seen(len, rows.y - rows.x, t - rows.x, p.causal, p.window);
  const int per = p.D / 32;
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int c = 0; c < per; ++c) q[c] = value_at(p.q, t * p.q_stride_t + h * p.q_stride_h + lane * per + c, p.dtype);
  for (int j = keys.x; j < keys.y; ++j) {
    const int page = p.page_table[b * p.table_stride + j / p.page_size];
    const bool there = page >= 0 && page < p.pages;
    const int64_t r = j % p.page_size;
    float s = 0.f;
    if (there)
      for (int c = 0; c < per; ++c)
        s += q[c] * value_at(p.key_cache, page * p.kc_stride_p + hk * p.kc_stride_h + r * p.kc_stride_r + lane * per + c, p.dtype);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= scale_log2;
    const float m_new = fmaxf(m, s);
    const float old = m == m_new ? 1.f : exp2f(m - m_new), e = exp2f(s - m_new);
    m = m_new;
    l = l * old + e;
    for (int c = 0; c < per; ++c) {
      const float v = there ? value_at(p.value_cache, page * p.vc_stride_p + hk * p.vc_stride_h + r * p.vc_stride_r + lane * per + c, p.dtype) : 0.f;
      acc[c] = acc[c] * old + e * v;
    }
  }
  const float inv = keys.y > keys.x ? 1.f / l : 0.f;
  for (int c = 0; c < per; ++c) put(p.o, t * p.o_stride_t + h * p.o_stride_h + lane * per + c, p.dtype, acc[c] * inv);
  if (p.lse != nullptr && lane == 0) p.lse[static_cast<int64_t>(t) * p.Hq + h] = keys.y > keys.x ? m + log2f(l) : -INFINITY;
}

// A warp per key of one head.
__global__ void __launch_bounds__(128) key_weights_rows_kernel(const __grid_constant__ dtb_paged_key_weights_params p, float scale_log2) {
  const int lane = threadIdx.x & 31, b = blockIdx.z, hk = blockIdx.y;
  const int64_t cap = static_cast<int64_t>(p.table_width) * p.page_size;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (j >= cap) return;
  const int len = table_len(p.kv_len, b, cap);
  float sum = 0.f;
  if (j < len) {
    const int2 rows = new_rows(p.query_start, b, p.T);
    const int page = p.page_table[b * p.table_stride + j / p.page_size];
    const bool there = page >= 0 && page < p.pages;
    const int64_t r = j % p.page_size;
    const int per = p.D / 32, G = p.Hq / p.Hkv;
    float k[4];
    for (int c = 0; c < per; ++c)
      k[c] = there ? value_at(p.key_cache, page * p.kc_stride_p + hk * p.kc_stride_h + r * p.kc_stride_r + lane * per + c, p.dtype) : 0.f;
    for (int t = rows.x; t < rows.y; ++t) {
      const int2 keys = seen(len, rows.y - rows.x, t - rows.x, p.causal, p.window);
      if (j < keys.x || j >= keys.y) continue;
      for (int g = 0; g < G; ++g) {
        const int h = hk * G + g;
        float s = 0.f;
        for (int c = 0; c < per; ++c) s += k[c] * value_at(p.q, t * p.q_stride_t + h * p.q_stride_h + lane * per + c, p.dtype);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        sum += exp2f(s * scale_log2 - p.lse[static_cast<int64_t>(t) * p.Hq + h]);
      }
    }
    if (p.prior != nullptr) sum += p.prior[b * p.prior_stride_b + hk * p.prior_stride_h + j];
  }
  if (lane == 0) p.out[b * p.out_stride_b + hk * p.out_stride_h + j] = sum;
}

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

extern "C" size_t dtb_paged_attn_workspace_bytes(const dtb_paged_attn_params* p) {
  (void)p;
  return 0;
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
  const float scale = p->scale > 0.f ? p->scale : 1.0f / sqrtf(static_cast<float>(p->D));
  const int64_t rows = static_cast<int64_t>(p->T) * p->Hq;
  paged_rows_kernel<<<static_cast<unsigned>((rows + 3) / 4), 128, 0, static_cast<cudaStream_t>(stream)>>>(*p, scale * kLog2e);
  (void)workspace;
  (void)workspace_bytes;
  return launch_ok("paged_rows_kernel launch") ? DTB_OK : DTB_ERR_LAUNCH;
}

extern "C" int dtb_paged_key_weights(const dtb_paged_key_weights_params* p, void* stream) {
  using namespace dtb;
  if (p == nullptr) return DTB_ERR_NULL;
  if (p->B == 0 || p->table_width == 0) return check_batch(p);
  if (p->key_cache == nullptr || p->out == nullptr || p->page_table == nullptr || p->query_start == nullptr || p->kv_len == nullptr)
    return DTB_ERR_NULL;
  if (p->T > 0 && (p->q == nullptr || p->lse == nullptr)) return DTB_ERR_NULL;    // without new tokens there are none to read
  if (const int st = check_batch(p)) return st;
  if (p->B > 65535 || p->Hkv > 65535) return DTB_ERR_SHAPE;
  const int64_t cap = static_cast<int64_t>(p->table_width) * p->page_size;
  const float scale = p->scale > 0.f ? p->scale : 1.0f / sqrtf(static_cast<float>(p->D));
  key_weights_rows_kernel<<<dim3(static_cast<unsigned>((cap + 3) / 4), p->Hkv, p->B), 128, 0, static_cast<cudaStream_t>(stream)>>>(*p, scale * kLog2e);
  return launch_ok("key_weights_rows_kernel launch") ? DTB_OK : DTB_ERR_LAUNCH;
}
