// Rotary positions of queries and keys, and the step in front of paged attention that uses them: new keys turned and
// written, with the values, into the pages of their sequences.
//
// A warp takes one token, or a part of its heads where tokens are few, and needs no other warp.  It asks for its first rows,
// makes the token's cosines and sines under them, two or so a lane, into its part of shared memory, and then goes over the
// rows, a unit of 2 V channels at a time: V at c0 and V at c1, half the turned channels behind, so that neighbouring lanes
// read neighbouring 16 bytes in both layouts.
//
// The angle in turns is taken in 64 bits, because a position of 10^6 times the fastest pair's frequency leaves no digit of a
// 32-bit product's fraction right, then reduced to half a turn and handed to sincospif with the part that 32 bits drop put
// back to first order.  Products and sums are f32, with one rounding at the end.
//
// Bound by bytes, each row read once and written once: 33792 tokens x 48 heads (830 MB) take 152 us, 5.5 TB/s.  A block a token,
// its threads waiting for each other between angles and rows, took 248 us; a warp a token with 80 registers, some of them
// spilled, 217.
#include <algorithm>

#include <cuda_fp16.h>

#include "host_common.h"
#include "paged.cuh"

namespace dtb {
namespace {

constexpr int kWarps = 4;        // of a block
constexpr int kAhead = 4;        // units of a lane that are asked for ahead
constexpr int kBlocks = 5;       // of an SM: 102 registers

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
  int first_head[3];               // of each tensor, among all
  int units;                       // of a row
  int lanes_log2;                  // lanes of a row, at most 32
  int parts, part_rows;            // warps of a token, and the rows (heads) that each takes
};

// V channels as loaded and stored, and as f32.
template <class E, int V> struct __align__(sizeof(E) * V) Vec {
  E x[V];
  __device__ __forceinline__ void up(float (&f)[V]) const {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = static_cast<float>(x[k]);
  }
  __device__ __forceinline__ void down(const float (&f)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = static_cast<E>(f[k]);
  }
};
template <int V> struct __align__(2 * V) Bf16Words {       // in pairs: a shift and a mask, and one rounding for both
  uint32_t x[V / 2];
  __device__ __forceinline__ void up(float (&f)[V]) const {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      f[2 * k] = __uint_as_float(x[k] << 16);
      f[2 * k + 1] = __uint_as_float(x[k] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void down(const float (&f)[V]) {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const __nv_bfloat162 w = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
      x[k] = *reinterpret_cast<const uint32_t*>(&w);
    }
  }
};
template <int V> struct __align__(2 * V) HalfWords {
  uint32_t x[V / 2];
  __device__ __forceinline__ void up(float (&f)[V]) const {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&x[k]));
      f[2 * k] = w.x;
      f[2 * k + 1] = w.y;
    }
  }
  __device__ __forceinline__ void down(const float (&f)[V]) {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const __half2 w = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
      x[k] = *reinterpret_cast<const uint32_t*>(&w);
    }
  }
};
template <class E, int V> struct VecOf { using T = Vec<E, V>; };
template <> struct VecOf<__nv_bfloat16, 8> { using T = Bf16Words<8>; };
template <> struct VecOf<__nv_bfloat16, 4> { using T = Bf16Words<4>; };
template <> struct VecOf<__nv_bfloat16, 2> { using T = Bf16Words<2>; };
template <> struct VecOf<__half, 8> { using T = HalfWords<8>; };
template <> struct VecOf<__half, 4> { using T = HalfWords<4>; };
template <> struct VecOf<__half, 2> { using T = HalfWords<2>; };

__device__ __forceinline__ double position_at(const void* p, int type, int64_t i) {
  if (type == 0) return static_cast<double>(static_cast<const int32_t*>(p)[i]);
  if (type == 1) return static_cast<double>(static_cast<const int64_t*>(p)[i]);
  return static_cast<double>(static_cast<const float*>(p)[i]);
}

// kHalf: pair i is channels (i, i + pairs), one at c0 and one at c1.  Else it is neighbours, at c0 or at c1.
// A lane keeps its place of the head and walks down the rows of all tensors, so that addresses are steps and the cosines and
// sines stay in registers; as soon as a row is written, the one kAhead passes on is asked for.
template <class E, int V, bool kHalf>
__global__ void __launch_bounds__(32 * kWarps, kBlocks) rotary_kernel(const __grid_constant__ RotaryKernelParams p) {
  extern __shared__ float2 cs_all[];                     // [warps][pairs] cosine and sine
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float2* cs = cs_all + warp * p.pairs;
  const uint32_t item = blockIdx.x * kWarps + warp;
  const uint32_t t = item / static_cast<uint32_t>(p.parts);
  if (t >= static_cast<uint32_t>(p.B) * p.S) return;     // whole warps; no barrier of the block follows
  const int part = static_cast<int>(item - t * p.parts);
  const int b = static_cast<int>(t / static_cast<uint32_t>(p.S)), s = static_cast<int>(t - static_cast<uint32_t>(b) * p.S);
  const int h_begin = part * p.part_rows, h_end = min(h_begin + p.part_rows, p.heads);
  const int turned = p.pairs / V;                        // units of a row that turn
  const int rest_half = ((p.D - 2 * p.pairs) / V + 1) >> 1;
  constexpr bool kNeighbours = !kHalf && V == 1;         // a pair's channels one by one
  using Vt = typename VecOf<E, V>::T;
  Vt x[kAhead], y[kAhead];
  float co[V], sn[V];

  const int rows = 32 >> p.lanes_log2;                   // rows of a warp's pass
  const int row = lane >> p.lanes_log2;
  int place = lane & ((1 << p.lanes_log2) - 1);          // unit of the row
  int c0 = 0, c1 = 0;
  auto at_place = [&]() {
    if (place < turned) {
      c0 = kNeighbours ? 2 * place : place * V;
      c1 = kNeighbours ? c0 + 1 : c0 + p.pairs;
    } else {
      c0 = 2 * p.pairs + (place - turned) * V;
      c1 = c0 + rest_half * V;
    }
  };
  at_place();
  // Rows are counted through the tensors: row h is of tensor w with first_head[w] <= h < first_head[w + 1].
  auto tensor_of = [&](int h) { return (h >= p.first_head[1]) + (h >= p.first_head[2]); };
  auto end_of = [&](int w) { return w == 0 ? p.first_head[1] : w == 1 ? p.first_head[2] : p.heads; };
  const E* in = nullptr;
  int64_t in_step = 0;
  int h_in = 0, in_end = 0;
  auto find_in = [&]() {                                 // where row h_in lies
    const int w = tensor_of(h_in);
    const RowsIn& r = p.t[w];
    in = reinterpret_cast<const E*>(r.in) + b * r.in_b + s * r.in_s + (h_in - p.first_head[w]) * r.in_h;
    in_step = rows * r.in_h;
    in_end = min(end_of(w), h_end);
  };
  auto start = [&]() {
    h_in = h_begin + row;
    if (h_in < h_end) find_in();
  };
  auto ask = [&](Vt& xi, Vt& yi) {
    if (h_in < h_end) {
      if (h_in >= in_end) find_in();
      xi = *reinterpret_cast<const Vt*>(in + c0);
      if (c1 < p.D) yi = *reinterpret_cast<const Vt*>(in + c1);
      in += in_step;
      h_in += rows;
    }
  };
  // the first rows are asked for ahead of everything else
  start();
  if (place < p.units) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ask(x[i], y[i]);
  }

  // Where the token goes, and its position.
  int64_t slot = 0;
  int page = -1;
  if (p.page_table != nullptr) {
    const int q = sequence_of(p.query_start, p.seqs, static_cast<int>(t));
    if (q < 0) return;                                   // a row of no sequence
    slot = static_cast<int64_t>(p.kv_len[q]) - p.query_start[q + 1] + t;
    const int64_t i = slot / p.page_size;
    if (p.pages > 0 && slot >= 0 && i < p.table_width) page = p.page_table[q * p.table_stride + i];
    if (page >= p.pages) page = -1;
  }
  for (int pair = lane; pair < p.pairs; pair += 32) {
    const int ax = p.axis != nullptr ? p.axis[pair] : 0;
    const double pos = p.positions != nullptr ? position_at(p.positions, p.pos_type, ax * p.pos_a + b * p.pos_b + s * p.pos_s)
                                              : static_cast<double>(slot);
    double turn = pos * p.turns[pair];
    turn -= rint(turn);
    const float hi = static_cast<float>(turn);
    const float lo = static_cast<float>(turn - hi) * 6.28318531f;
    float sine, cosine;
    sincospif(2.0f * hi, &sine, &cosine);
    cs[pair] = make_float2((cosine - sine * lo) * p.amplitude, (sine + cosine * lo) * p.amplitude * p.sign);
  }
  __syncwarp();
  const int64_t page_row = page >= 0 ? slot % p.page_size : 0;

  bool asked = true;
  for (; place < p.units; place += 32, asked = false) {  // heads of more than 32 units: again, further right
    at_place();
    if (!asked) {
      start();
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ask(x[i], y[i]);
    }
    const bool turns = place < turned;
    // in halves the pairs c0 .. ; as neighbours those of the V channels at c0 and then of the V at c1
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int pair = kHalf || kNeighbours ? place * V + k : (k < V / 2 ? (c0 >> 1) + k : (c1 >> 1) + k - V / 2);
      const float2 z = turns ? cs[pair] : make_float2(1.f, 0.f);
      co[k] = z.x;
      sn[k] = z.y;
    }
    E* out = nullptr;
    int64_t out_step = 0;
    bool writes = false, turn = false;
    for (int h = h_begin + row, out_end = 0; h < h_end;) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (h < h_end) {
          if (h >= out_end) {
            const int w = tensor_of(h);
            const RowsIn& r = p.t[w];
            out = reinterpret_cast<E*>(r.out) + (h - p.first_head[w]) * r.out_h + (r.paged ? page * r.out_b + page_row * r.out_s : b * r.out_b + s * r.out_s);
            out_step = rows * r.out_h;
            out_end = min(end_of(w), h_end);
            writes = !r.paged || page >= 0;
            turn = turns && r.turn;
          }
          if (turn) {
            float f[V], g[V], u[V], v[V];
            x[i].up(f);
            y[i].up(g);
            if constexpr (kHalf || kNeighbours) {
#pragma unroll
              for (int k = 0; k < V; ++k) {
                u[k] = f[k] * co[k] - g[k] * sn[k];
                v[k] = f[k] * sn[k] + g[k] * co[k];
              }
            } else {
#pragma unroll
              for (int k = 0; k < V / 2; ++k) {
                const int e0 = 2 * k, e1 = 2 * k + 1, m = k + V / 2;
                u[e0] = f[e0] * co[k] - f[e1] * sn[k];
                u[e1] = f[e0] * sn[k] + f[e1] * co[k];
                v[e0] = g[e0] * co[m] - g[e1] * sn[m];
                v[e1] = g[e0] * sn[m] + g[e1] * co[m];
              }
            }
            x[i].down(u);
            y[i].down(v);
          }
          if (writes) {
            *reinterpret_cast<Vt*>(out + c0) = x[i];
            if (c1 < p.D) *reinterpret_cast<Vt*>(out + c1) = y[i];
          }
          out += out_step;
          h += rows;
          ask(x[i], y[i]);
        }
      }
    }
  }
}

template <class E, int V>
int launch_v(const RotaryKernelParams& p, unsigned blocks, size_t smem, cudaStream_t s) {
  if (p.interleaved) rotary_kernel<E, V, false><<<blocks, 32 * kWarps, smem, s>>>(p);
  else rotary_kernel<E, V, true><<<blocks, 32 * kWarps, smem, s>>>(p);
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
  p.heads = p.t[0].heads + p.t[1].heads + p.t[2].heads;
  p.first_head[1] = p.t[0].heads;
  p.first_head[2] = p.t[0].heads + p.t[1].heads;
  p.units = p.pairs / v + ((p.D - 2 * p.pairs) / v + 1) / 2;
  while (p.lanes_log2 < 5 && 1 << p.lanes_log2 < p.units) ++p.lanes_log2;
  // Few tokens: as many warps a token as have work for one round each, up to some 24 a SM.
  const int64_t total = static_cast<int64_t>(p.B) * p.S;
  const int64_t rounds = ((static_cast<int64_t>(p.heads) << p.lanes_log2) + 32 * kAhead - 1) / (32 * kAhead);
  const int64_t parts = std::min<int64_t>({rounds, p.heads, std::max<int64_t>(148 * 24 / total, 1)});
  p.part_rows = static_cast<int>((p.heads + parts - 1) / parts);
  p.parts = (p.heads + p.part_rows - 1) / p.part_rows;
  const int64_t blocks = (total * p.parts + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffff / kWarps) return DTB_ERR_SHAPE;
  const size_t smem = static_cast<size_t>(kWarps) * p.pairs * sizeof(float2);
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
