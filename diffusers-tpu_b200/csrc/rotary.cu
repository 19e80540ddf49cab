// Rotary positions of queries and keys, and the step in front of paged attention that uses them: new keys turned and
// written, with the values, into the pages of their sequences.
//
// A thread keeps one place of the head (V pairs of channels, or V channels that are only copied) of one token and walks
// the heads of all tensors, so that the cosines and sines, which depend on the token and the pair alone, stay in
// registers.  A block's threads first make them together: the angle in turns is taken in 64 bits, because a position of
// 10^6 times the fastest pair's frequency leaves no digit of a 32-bit product's fraction right, then reduced to half a
// turn and handed to sincospif with the part that 32 bits drop put back to first order.  Products and sums are f32, with
// one rounding at the end.
#include <algorithm>

#include <cuda_fp16.h>

#include "host_common.h"
#include "paged.cuh"

namespace dtb {
namespace {

constexpr int kThreads = 256;

struct RowsIn {
  const char* in;
  int64_t in_b, in_s, in_h;        // element strides of an input row
  char* out;
  int64_t out_b, out_s, out_h;     // of an output row; a cache: (unused, row of a page, head), and out_b is the page's
  int heads;
  int turn, paged;
};

struct RotaryKernelParams {
  RowsIn t[3];
  const double* turns;
  const int32_t* axis;
  const void* positions;
  int64_t pos_a, pos_b, pos_s;
  const int32_t* page_table;
  const int32_t* query_start;
  const int32_t* kv_len;
  int64_t table_stride;
  int table_width, pages, page_size, seqs;
  int pos_type, B, S, D, pairs, heads, interleaved;
  float amplitude, sign;
  int places;                      // threads of a row
  int rows;                        // rows (heads) that a token's threads hold at a time
  int tokens;                      // tokens of a block
};

template <class E> struct Cvt;
template <> struct Cvt<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Cvt<__half> {
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct Cvt<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};

template <class E, int V> struct __align__(sizeof(E) * V) Vec { E x[V]; };

__device__ __forceinline__ double position_at(const void* p, int type, int64_t i) {
  if (type == 0) return static_cast<double>(static_cast<const int32_t*>(p)[i]);
  if (type == 1) return static_cast<double>(static_cast<const int64_t*>(p)[i]);
  return static_cast<double>(static_cast<const float*>(p)[i]);
}

// kHalf: pair i is channels (i, i + pairs): a place is V channels and their V partners.  Else a place is 2 V neighbours.
template <class E, int V, bool kHalf>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryKernelParams p) {
  extern __shared__ float2 cs[];                         // [tokens][pairs] cosine and sine
  __shared__ int64_t slot_of[kThreads];                  // slot of a token in its sequence, -1 = none
  __shared__ int page_of[kThreads];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tokens;
  const int64_t total = static_cast<int64_t>(p.B) * p.S;
  const bool cached = p.page_table != nullptr;
  if (cached) {
    if (threadIdx.x < p.tokens) {
      const int64_t t = first + threadIdx.x;
      int64_t slot = -1;
      int page = -1;
      const int b = t < total ? sequence_of(p.query_start, p.seqs, static_cast<int>(t)) : -1;
      if (b >= 0) {
        slot = static_cast<int64_t>(p.kv_len[b]) - p.query_start[b + 1] + t;
        const int64_t i = slot / p.page_size;
        if (slot >= 0 && i < p.table_width) page = p.page_table[b * p.table_stride + i];
        if (page < 0 || page >= p.pages) page = -1;
      }
      slot_of[threadIdx.x] = slot;
      page_of[threadIdx.x] = b >= 0 ? page : -2;         // -2: a row of no sequence
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < p.tokens * p.pairs; i += kThreads) {
    const int tk = i / p.pairs, pair = i - tk * p.pairs;
    const int64_t t = first + tk;
    if (t >= total) continue;
    const int64_t b = t / p.S, s = t - b * p.S;
    const int ax = p.axis != nullptr ? p.axis[pair] : 0;
    const double pos = p.positions != nullptr ? position_at(p.positions, p.pos_type, ax * p.pos_a + b * p.pos_b + s * p.pos_s)
                                              : static_cast<double>(slot_of[tk]);
    double turn = pos * p.turns[pair];
    turn -= rint(turn);
    const float hi = static_cast<float>(turn);
    const float lo = static_cast<float>(turn - hi) * 6.28318531f;
    float sn, co;
    sincospif(2.0f * hi, &sn, &co);
    cs[i] = make_float2((co - sn * lo) * p.amplitude, (sn + co * lo) * p.amplitude * p.sign);
  }
  __syncthreads();

  const int per_token = p.places * p.rows;
  const int tk = threadIdx.x / per_token;
  const int64_t t = first + tk;
  if (tk >= p.tokens || t >= total) return;
  const int64_t b = t / p.S, s = t - b * p.S;
  const int page = cached ? page_of[tk] : 0;
  if (page == -2) return;
  const int64_t page_row = cached ? slot_of[tk] % p.page_size : 0;
  const int in_token = threadIdx.x - tk * per_token;
  const int row0 = in_token / p.places, place = in_token - row0 * p.places;
  // Channels of this place: V at c0 and V at c1.
  const int turned = p.pairs / V;                        // places that turn
  const bool turns = place < turned;
  int c0, c1;
  if (turns) {
    c0 = kHalf ? place * V : place * 2 * V;
    c1 = kHalf ? c0 + p.pairs : c0 + V;
  } else {
    c0 = 2 * p.pairs + (place - turned) * 2 * V;
    c1 = c0 + V;
  }
  const bool second = c1 + V <= p.D;
  float co[V], sn[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 x = turns ? cs[tk * p.pairs + place * V + i] : make_float2(1.f, 0.f);
    co[i] = x.x;
    sn[i] = x.y;
  }
  using Vt = Vec<E, V>;
  for (int h = row0; h < p.heads; h += p.rows) {
    int which = 0, head = h;
    if (head >= p.t[0].heads) { head -= p.t[0].heads; which = 1; }
    if (which == 1 && head >= p.t[1].heads) { head -= p.t[1].heads; which = 2; }
    const RowsIn& r = p.t[which];
    if (r.paged && page < 0) continue;
    const E* in = reinterpret_cast<const E*>(r.in) + b * r.in_b + s * r.in_s + head * r.in_h;
    E* out = reinterpret_cast<E*>(r.out) + head * r.out_h +
             (r.paged ? static_cast<int64_t>(page) * r.out_b + page_row * r.out_s : b * r.out_b + s * r.out_s);
    Vt x = *reinterpret_cast<const Vt*>(in + c0), y = x;
    if (second) y = *reinterpret_cast<const Vt*>(in + c1);
    if (turns && r.turn) {
      Vt xo, yo;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // pair i of the place: (x[i], y[i]) with halves, neighbours 2i and 2i + 1 of x | y otherwise
        const int e0 = 2 * i, e1 = 2 * i + 1;
        const float a = Cvt<E>::up(kHalf ? x.x[i] : (e0 < V ? x.x[e0 % V] : y.x[e0 % V]));
        const float c = Cvt<E>::up(kHalf ? y.x[i] : (e1 < V ? x.x[e1 % V] : y.x[e1 % V]));
        const E ra = Cvt<E>::down(a * co[i] - c * sn[i]);
        const E rc = Cvt<E>::down(a * sn[i] + c * co[i]);
        if (kHalf) {
          xo.x[i] = ra;
          yo.x[i] = rc;
        } else {
          (e0 < V ? xo : yo).x[e0 % V] = ra;
          (e1 < V ? xo : yo).x[e1 % V] = rc;
        }
      }
      x = xo;
      y = yo;
    }
    *reinterpret_cast<Vt*>(out + c0) = x;
    if (second) *reinterpret_cast<Vt*>(out + c1) = y;
  }
}

template <class E, int V>
int launch_v(const RotaryKernelParams& p, unsigned blocks, size_t smem, cudaStream_t s) {
  if (p.interleaved) rotary_kernel<E, V, false><<<blocks, kThreads, smem, s>>>(p);
  else rotary_kernel<E, V, true><<<blocks, kThreads, smem, s>>>(p);
  return launch_ok("rotary_kernel launch") ? DTB_OK : DTB_ERR_LAUNCH;
}

// Widest access, in elements, that every row of the call allows: pairs and the rest of the head are whole vectors, and
// pointers and strides are multiples of it.
int widest(const RotaryKernelParams& p, int esz) {
  for (int v = 16 / esz; v > 1; v /= 2) {
    bool ok = p.pairs % v == 0 && p.D % v == 0;
    for (const RowsIn& r : p.t) {
      if (r.heads == 0) continue;
      const int64_t bytes = static_cast<int64_t>(v) * esz;
      ok = ok && reinterpret_cast<uintptr_t>(r.in) % bytes == 0 && reinterpret_cast<uintptr_t>(r.out) % bytes == 0;
      for (int64_t st : {r.in_b, r.in_s, r.in_h, r.out_b, r.out_s, r.out_h}) ok = ok && st % v == 0;
    }
    if (ok) return v;
  }
  return 1;
}

int launch(RotaryKernelParams& p, int dtype, cudaStream_t s) {
  const int esz = dtype == DTB_FP32 ? 4 : 2;
  const int v = widest(p, esz);
  // places of 2 V channels; the last of the copied ones may be half empty
  p.places = p.pairs / v + (p.D - 2 * p.pairs + 2 * v - 1) / (2 * v);
  if (p.places > kThreads) return DTB_ERR_SHAPE;
  p.heads = p.t[0].heads + p.t[1].heads + p.t[2].heads;
  p.rows = std::min(p.heads, kThreads / p.places);
  p.tokens = std::max(1, kThreads / (p.places * p.rows));
  const int64_t total = static_cast<int64_t>(p.B) * p.S;
  // no more tokens a block than keep all SMs busy
  while (p.tokens > 1 && total / p.tokens < 148) p.tokens /= 2;
  const int64_t blocks = (total + p.tokens - 1) / p.tokens;
  if (blocks > 0x7fffffff) return DTB_ERR_SHAPE;
  const size_t smem = static_cast<size_t>(p.tokens) * p.pairs * sizeof(float2);
  if (smem > 40000) return DTB_ERR_SHAPE;
  const unsigned n = static_cast<unsigned>(blocks);
  if (dtype == DTB_FP32) {
    if (v == 4) return launch_v<float, 4>(p, n, smem, s);
    if (v == 2) return launch_v<float, 2>(p, n, smem, s);
    return launch_v<float, 1>(p, n, smem, s);
  }
  if (dtype == DTB_FP16) {
    if (v == 8) return launch_v<__half, 8>(p, n, smem, s);
    if (v == 4) return launch_v<__half, 4>(p, n, smem, s);
    if (v == 2) return launch_v<__half, 2>(p, n, smem, s);
    return launch_v<__half, 1>(p, n, smem, s);
  }
  if (v == 8) return launch_v<__nv_bfloat16, 8>(p, n, smem, s);
  if (v == 4) return launch_v<__nv_bfloat16, 4>(p, n, smem, s);
  if (v == 2) return launch_v<__nv_bfloat16, 2>(p, n, smem, s);
  return launch_v<__nv_bfloat16, 1>(p, n, smem, s);
}

constexpr int kMaxDim = 512;

int check_rotation(int D, int rotary, int n_axes, int pos_type, const int32_t* axis) {
  if (D <= 0 || D > kMaxDim || rotary < 0 || rotary > D || rotary % 2 != 0) return DTB_ERR_SHAPE;
  if (n_axes <= 0 || (n_axes > 1 && axis == nullptr)) return DTB_ERR_SHAPE;
  if (pos_type < 0 || pos_type > 2) return DTB_ERR_DTYPE;
  return DTB_OK;
}

}  // namespace
}  // namespace dtb

extern "C" int dtb_rotary(const dtb_rotary_params* rp, void* stream) {
  using namespace dtb;
  if (rp == nullptr || rp->q == nullptr || rp->q_out == nullptr || rp->turns == nullptr || rp->positions == nullptr) return DTB_ERR_NULL;
  if ((rp->k == nullptr) != (rp->k_out == nullptr)) return DTB_ERR_NULL;
  if (rp->dtype < 0 || rp->dtype > DTB_FP32) return DTB_ERR_DTYPE;
  if (rp->B < 0 || rp->S < 0 || rp->Hq <= 0 || rp->Hk < 0 || (rp->k != nullptr && rp->Hk == 0)) return DTB_ERR_SHAPE;
  if (const int st = check_rotation(rp->D, rp->rotary, rp->n_axes, rp->pos_type, rp->axis)) return st;
  if (rp->rotary == 0) return DTB_ERR_SHAPE;
  if (rp->B == 0 || rp->S == 0) return DTB_OK;
  RotaryKernelParams p = {};
  p.t[0] = {static_cast<const char*>(rp->q), rp->q_stride_b, rp->q_stride_s, rp->q_stride_h,
            static_cast<char*>(rp->q_out), rp->qo_stride_b, rp->qo_stride_s, rp->qo_stride_h, rp->Hq, 1, 0};
  if (rp->k != nullptr)
    p.t[1] = {static_cast<const char*>(rp->k), rp->k_stride_b, rp->k_stride_s, rp->k_stride_h,
              static_cast<char*>(rp->k_out), rp->ko_stride_b, rp->ko_stride_s, rp->ko_stride_h, rp->Hk, 1, 0};
  p.turns = rp->turns;
  p.axis = rp->axis;
  p.positions = rp->positions;
  p.pos_a = rp->pos_stride_a;
  p.pos_b = rp->pos_stride_b;
  p.pos_s = rp->pos_stride_s;
  p.pos_type = rp->pos_type;
  p.B = rp->B;
  p.S = rp->S;
  p.D = rp->D;
  p.pairs = rp->rotary / 2;
  p.interleaved = rp->interleaved;
  p.amplitude = rp->amplitude;
  p.sign = rp->transpose ? -1.0f : 1.0f;
  return launch(p, rp->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int dtb_paged_append(const dtb_paged_append_params* ap, void* stream) {
  using namespace dtb;
  if (ap == nullptr || ap->k == nullptr || ap->v == nullptr || ap->key_cache == nullptr || ap->value_cache == nullptr ||
      ap->page_table == nullptr || ap->query_start == nullptr || ap->kv_len == nullptr)
    return DTB_ERR_NULL;
  if ((ap->q == nullptr) != (ap->q_out == nullptr)) return DTB_ERR_NULL;
  if (ap->dtype != DTB_BF16 && ap->dtype != DTB_FP16) return DTB_ERR_DTYPE;
  if (ap->B < 0 || ap->T < 0 || ap->Hkv <= 0 || ap->Hq < 0 || (ap->q != nullptr && ap->Hq == 0)) return DTB_ERR_SHAPE;
  if (ap->pages < 0 || ap->page_size <= 0 || ap->table_width < 0) return DTB_ERR_SHAPE;
  const int rotary = ap->turns != nullptr ? ap->rotary : 0;
  if (ap->turns != nullptr && rotary == 0) return DTB_ERR_SHAPE;
  if (const int st = check_rotation(ap->D, rotary, ap->n_axes, ap->pos_type, ap->axis)) return st;
  if (ap->n_axes > 1 && ap->positions == nullptr) return DTB_ERR_NULL;     // a slot is one position
  if (ap->B == 0 || ap->T == 0) return DTB_OK;
  RotaryKernelParams p = {};
  if (ap->q != nullptr)
    p.t[0] = {static_cast<const char*>(ap->q), 0, ap->q_stride_t, ap->q_stride_h,
              static_cast<char*>(ap->q_out), 0, ap->qo_stride_t, ap->qo_stride_h, ap->Hq, 1, 0};
  p.t[1] = {static_cast<const char*>(ap->k), 0, ap->k_stride_t, ap->k_stride_h,
            static_cast<char*>(ap->key_cache), ap->kc_stride_p, ap->kc_stride_r, ap->kc_stride_h, ap->Hkv, 1, 1};
  p.t[2] = {static_cast<const char*>(ap->v), 0, ap->v_stride_t, ap->v_stride_h,
            static_cast<char*>(ap->value_cache), ap->vc_stride_p, ap->vc_stride_r, ap->vc_stride_h, ap->Hkv, 0, 1};
  p.turns = ap->turns;
  p.axis = ap->axis;
  p.positions = ap->positions;
  p.pos_a = ap->pos_stride_a;
  p.pos_s = ap->pos_stride_t;
  p.pos_type = ap->pos_type;
  p.page_table = ap->page_table;
  p.query_start = ap->query_start;
  p.kv_len = ap->kv_len;
  p.table_stride = ap->table_stride;
  p.table_width = ap->table_width;
  p.pages = ap->pages;
  p.page_size = ap->page_size;
  p.seqs = ap->B;
  p.B = 1;
  p.S = ap->T;
  p.D = ap->D;
  p.pairs = rotary / 2;
  p.interleaved = ap->interleaved;
  p.amplitude = ap->amplitude;
  p.sign = 1.0f;
  return launch(p, ap->dtype, static_cast<cudaStream_t>(stream));
}
