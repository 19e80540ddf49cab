// Attention of new tokens over a paged key/value cache, for sm_100a.
//
// Rows.  A key head's query rows are its group's heads of each new token: row r of a 128-row tile is head r % G of token
// r / G, so a tile holds 128 / G tokens (whole ones), one TMA box of [tokens, G, 64 channels] fills it, and a decode step
// of one token still has G rows to show the tensor core.  A query block is two such tiles that share the keys; the second is
// left out where the block's tokens fit the first.
//
// Loop.  S = Q K^T on tcgen05 into tensor memory, a softmax thread per row with the running maximum and sum in registers,
// P beside S in the inputs' type, O += P V: the warp roles, the tensor memory and the order between the warps are those of
// attn_kernel.cuh, here carried over many units of work a block (paged_plan.cuh) by running counts of each barrier's uses.
// K and V tiles of 128 keys come through a ring of 160 KB, as 128 / page_size boxes a tile and 64 channels, each lane of the
// producer warp issuing one of them; pages outside the cache and keys that no row of the block sees are fetched from past its
// end, where TMA writes zeros.
//
// Units of few rows.  Where a block's rows are 16 at most (single tokens, mostly) the keys are the 128 rows instead: S^T =
// K Q^T and O^T += V^T P^T with 16 columns, a softmax thread a key, P written to shared memory (the second query tile's,
// which such units have no use for).  Padding few rows to 128 costs no time while the clock is up, but eight times the
// products: 48 single tokens over 2000-32768 keys x 8 heads ran into the power limit within 30 ms, and then took 425 us for
// 355.  A thread's share of the sum stays in registers until the end; the maximum is agreed on only in tiles where some thread
// found a logit 2^8 above the one in use, by one vote a tile of the four warps.
//
// Masks.  A row sees keys [lo, hi) of its sequence; tiles that reach out of some row's are masked by column with -inf.  P = 0
// does not stop a NaN among V's rows, so V rows that no row of the block sees and that lie in a fetched page (the end of a
// sequence's last page is whatever was there) are zeroed in shared memory before the product.
//
// Roundings: S, the maximum, the sum and O are f32; P is rounded to the inputs' type, as the tensor core takes no other;
// the result is rounded once.  With fp16 the offset of the exponentials stays 7 below the running maximum, so that P reaches
// 2^15 and what falls below fp16's smallest number is a 2^-39 part of the row's largest.
#pragma once

#include <type_traits>

#include <cuda_fp16.h>

#include "paged_plan.cuh"

namespace dtb {

constexpr int kBlockM = 128, kBlockN = kPlanTile;  // query rows and keys of a tile
constexpr uint32_t kPanelBytes = 128 * 64 * 2;
constexpr int kMmaWarp = 8, kLoadWarp = 9, kPvWarp = 10;     // warps 0-3 and 4-7: softmax of the two query tiles; 11: units
constexpr int kPagedThreads = kPlanThreads;
static_assert(kPagedThreads == 384, "three warpgroups");
// Register hand-over between warpgroups, as in attn_kernel.cuh: an inc that asks for more than the decs released waits for
// ever, so the launch refuses a build that was not compiled for kLaunchRegs.
constexpr int kLaunchRegs = 168, kRegsSoftmax = 224, kRegsService = 56;
static_assert((kLaunchRegs - kRegsService) * 128 >= (kRegsSoftmax - kLaunchRegs) * 256, "setmaxnreg.inc would ask for more registers than are released");
static_assert(kPagedThreads * kLaunchRegs <= 65536, "the CTA does not fit the register file");
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleThreshold = 8.0f;    // log2 units: O is rescaled only when the row maximum grew by more than 2^8
constexpr float kLowestOffset = -3.402823466e38f;   // the largest finite float, negated: below the maximum of any row that has one
constexpr int kRingBytes = 5 * 32768;      // with two query tiles of 32 KB and the barriers, all that a block can have
constexpr int kThinRows = 16;                // rows of a unit that is computed with keys as rows
constexpr uint32_t kThinPanel = kThinRows * 128;     // its P: two panels of 64 keys, then what the four warps tell each other
constexpr uint32_t kThinTop = 2 * kThinPanel, kThinSum = kThinTop + 4 * kThinRows * 4, kThinVotes = kThinSum + 4 * kThinRows * 4;
static_assert(kThinVotes + 8 * 4 <= kPanelBytes, "P and the exchange lie in the second query tile");
constexpr int kSegs = 16;                    // units whose description is held at a time

// Of a unit swept in pieces: what the merge needs, written by the block that has the first piece.
struct __align__(16) MergeDesc {
  int pieces;                // 0: nothing to merge
  int tok0, ntok, hk;
};

constexpr int kSlotRows = 256;
template <int kD> constexpr size_t kSlotFloats = static_cast<size_t>(kSlotRows) * (kD + 2);

struct PagedKernelParams {
  CUtensorMap tmap_q, tmap_k, tmap_v;
  PlanParams plan;
  const int32_t* page_table;
  int64_t table_stride;
  int table_width, pages, page_size;
  void* o;
  int64_t o_stride_t, o_stride_h;
  float* lse;
  float* slots;              // [2 * blocks] of kSlotFloats: O, then m, then l
  MergeDesc* merge;          // [blocks]
  int32_t* status;
  int Hq, G, tile_tokens;    // G heads a group, 128 / G tokens a tile
  float scale_log2;
};

template <int kD>
struct __align__(8) PagedBarriers {
  static constexpr int kSlots = kRingBytes / (128 * kD * 2);
  uint64_t q_full, q_empty;
  uint64_t kv_full[kSlots], kv_empty[kSlots];
  uint64_t s_full[2], p_lo[2], p_hi[2], pv_done[2];
  uint64_t o_free[2][2];     // of each group, its units with keys in turn: see o_free_of
  uint64_t s_free, vote;
  uint64_t seg_full[kSegs], seg_empty[kSegs];
  uint32_t tmem_base;
  int abort_flag;
  Seg segs[kSegs];           // a ring: the plan fills the first kSegs units' places, the idle warp the others'
  BlockUnits units;
};

template <int kD>
constexpr size_t kPagedSmem = 1024 + 2 * 128 * kD * 2 + kRingBytes + sizeof(PagedBarriers<kD>);
static_assert(kPagedSmem<128> <= 232448, "more shared memory than a block can have");

enum PagedSite : int { SITE_PG_Q = 110, SITE_PG_QE = 111, SITE_PG_KV = 120, SITE_PG_KVE = 130, SITE_PG_S = 140, SITE_PG_P = 150, SITE_PG_PH = 155,
                       SITE_PG_O = 160, SITE_PG_SF = 165, SITE_PG_OF = 170, SITE_PG_END = 180, SITE_PG_SEG = 190, SITE_PG_SEGE = 195, SITE_PG_VOTE = 200 };

// Where unit n (counted among a group's units with keys) says that it is over, and the parity of that.  The units take two barriers
// in turn because the producer asks about the unit before the one that it loads: with Q of that unit read the one two before it is
// over, and the one behind it has not begun, so each parity of a barrier names one unit however late the producer comes; on a
// barrier for all units it names the unit before or the one before that.
template <class Bars>
__device__ __forceinline__ uint64_t* o_free_of(Bars* bars, int t, int n) { return &bars->o_free[t][n & 1]; }
__device__ __forceinline__ uint32_t o_free_parity(int n) { return (n >> 1) & 1; }

// Warp-uniform bounded wait: every lane polls, and the warp agrees on the outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const AbortCtx& ctx, int site) {
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, ctx, site));
}

// Division by a small constant of the launch: q = n / d for 0 <= n < 2^16.
__device__ __forceinline__ int div_small(int n, uint32_t magic) { return static_cast<int>((static_cast<uint32_t>(n) * magic) >> 16); }

template <class E> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <class E> constexpr float kOffsetBelowMax = 0.f;
template <> constexpr float kOffsetBelowMax<__half> = 7.f;

template <class E> __host__ __device__ constexpr uint32_t paged_idesc(int n, bool b_mn_major) {
  return make_idesc_bf16(128, n, false, b_mn_major) & (sizeof(E) && std::is_same<E, __half>::value ? ~((7u << 7) | (7u << 10)) : ~0u);
}

constexpr int kSegReaders = 11;              // warps that take the units: producer, both issuers, eight of softmax

// One key tile of softmax for the row of this thread, of which columns [lo, hi) count.  As softmax_tile of attn_kernel.cuh.
template <class E, int kD, class WaitPv>
__device__ __forceinline__ bool paged_softmax_tile(uint32_t s_tmem, uint32_t p_tmem, uint32_t o_tmem, float scale_log2, bool masked, int lo, int hi,
                                                   bool o_live, float& m_used, float& l_sum, uint32_t bar_s_free, uint32_t bar_p_lo,
                                                   uint32_t bar_p_hi, WaitPv wait_pv) {
  uint32_t sr[kBlockN];
  tmem_ld128_sync(s_tmem, sr);
  tc_fence_before();
  mbar_arrive(bar_s_free);
  if (masked) {
#pragma unroll
    for (int i = 0; i < kBlockN; ++i)
      if (i >= hi || i < lo) sr[i] = 0xff800000u;  // -inf
  }
  const uint64_t scale2 = pack_f32x2(scale_log2, scale_log2);
  uint64_t acc2 = pack_f32x2(0.f, 0.f);
  uint32_t pk[32];
  auto exp_half = [&](int half) {
    const uint64_t neg_m2 = pack_f32x2(-m_used, -m_used);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int col = half * 64 + 2 * i;
      const uint64_t x2 = fma_f32x2(pack_f32x2(__uint_as_float(sr[col]), __uint_as_float(sr[col + 1])), scale2, neg_m2);
      float x0, x1;
      unpack_f32x2(x2, x0, x1);
      const float p0 = ex2(x0), p1 = ex2(x1);
      acc2 = add_f32x2(acc2, pack_f32x2(p0, p1));
      pk[i] = pack2<E>(p0, p1);
      if (i == 15) tmem_st16(p_tmem + half * 32, pk);
    }
  };
  auto publish = [&](int half) {
    tmem_st16(p_tmem + half * 32 + 16, pk + 16);
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(half == 0 ? bar_p_lo : bar_p_hi);
  };
  if (!wait_pv()) return false;
  float mxs[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) mxs[c] = fmaxf(__uint_as_float(sr[c]), __uint_as_float(sr[c + 8]));
#pragma unroll
  for (int i = 16; i < kBlockN; i += 16) {
#pragma unroll
    for (int c = 0; c < 8; ++c) mxs[c] = max3(mxs[c], __uint_as_float(sr[i + c]), __uint_as_float(sr[i + c + 8]));
  }
  const float mx = fmaxf(max3(mxs[0], mxs[1], mxs[2]), fmaxf(max3(mxs[3], mxs[4], mxs[5]), fmaxf(mxs[6], mxs[7]))) * scale_log2 - kOffsetBelowMax<E>;
  const bool grow = mx > m_used + kRescaleThreshold;   // always, for a finite maximum, while m_used is kLowestOffset
  if (o_live && __any_sync(0xffffffffu, grow)) {
    const float alpha = grow ? ex2(m_used - mx) : 1.0f;
    l_sum *= alpha;
    uint32_t r[32];
#pragma unroll
    for (int c = 0; c < kD / 32; ++c) {
      tmem_ld32_sync(o_tmem + c * 32, r);
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
      tmem_st32(o_tmem + c * 32, r);
    }
  }
  if (grow) m_used = mx;
  exp_half(0);
  publish(0);
  exp_half(1);
  publish(1);
  float a0, a1;
  unpack_f32x2(acc2, a0, a1);
  l_sum += a0 + a1;
  return true;
}

// 16 consecutive columns of tensor memory, with the wait.
__device__ __forceinline__ void tmem_ld16_sync(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// What the four warps of a softmax group tell each other, through a barrier whose waits are bounded as all others are.
struct ThinGroup {
  uint64_t* bar;             // one arrival a warp
  uint8_t* thin;             // P, then what is exchanged
  int turns;                 // of the barrier so far
  __device__ __forceinline__ float* top() const { return reinterpret_cast<float*>(thin + kThinTop); }      // [warp][column]
  __device__ __forceinline__ float* sums() const { return reinterpret_cast<float*>(thin + kThinSum); }
  __device__ __forceinline__ bool sync(const AbortCtx& ctx) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(bar));
    return warp_wait(bar, turns++ & 1, ctx, SITE_PG_VOTE);
  }
  // `any`: x holds in some thread of the group.  Two places in turn: one may still be read when the next vote is written.
  __device__ __forceinline__ bool vote(bool x, const AbortCtx& ctx, bool& any) {
    int* votes = reinterpret_cast<int*>(thin + kThinVotes) + (turns & 1) * 4;
    x = __any_sync(0xffffffffu, x);
    if ((threadIdx.x & 31) == 0) votes[(threadIdx.x >> 5) & 3] = x;
    if (!sync(ctx)) return false;
    const volatile int* v = votes;
    any = (v[0] | v[1] | v[2] | v[3]) != 0;
    return true;
  }
};

// f(c) for the columns in use, eight at a time.
template <class F>
__device__ __forceinline__ void thin_columns(int cols, F f) {
#pragma unroll
  for (int c = 0; c < 8; ++c) f(c);
  if (cols > 8) {
#pragma unroll
    for (int c = 8; c < kThinRows; ++c) f(c);
  }
}

// One key tile of softmax with the key of this thread as row: columns [lo, hi) see it.  m is the same in all threads, l the
// part of this thread's keys.
template <class E, class WaitPv>
__device__ __forceinline__ bool thin_softmax_tile(uint32_t s_tmem, uint32_t o_tmem, ThinGroup& group, const AbortCtx& ctx, float scale_log2, int cols, int lo, int hi,
                                                  bool o_live, float (&m)[kThinRows], float (&l)[kThinRows], uint32_t bar_s_free, uint32_t bar_p_lo,
                                                  uint32_t bar_p_hi, WaitPv wait_pv) {
  const int r = threadIdx.x & (kBlockM - 1), warp = r >> 5, lane = r & 31;
  uint32_t sr[kThinRows];
  tmem_ld16_sync(s_tmem, sr);
  tc_fence_before();
  mbar_arrive(bar_s_free);
  bool grow = false;
  thin_columns(cols, [&](int c) {
    if (c < lo || c >= hi) sr[c] = 0xff800000u;          // -inf; columns behind the last too
    grow |= fmaf(__uint_as_float(sr[c]), scale_log2, -m[c]) > kRescaleThreshold + kOffsetBelowMax<E>;
  });
  bool any = false;
  if (!group.vote(grow, ctx, any) || !wait_pv()) return false;
  if (any) {
    float* top = group.top();
    float mine = -INFINITY;
    thin_columns(cols, [&](int c) {
      float x = __uint_as_float(sr[c]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
      if (lane == c) mine = x;
    });
    if (lane < kThinRows) top[warp * kThinRows + lane] = mine;
    if (!group.sync(ctx)) return false;
    uint32_t o[kThinRows];
    if (o_live) tmem_ld16_sync(o_tmem, o);
    thin_columns(cols, [&](int c) {
      const float mx = fmaxf(fmaxf(top[c], top[kThinRows + c]), fmaxf(top[2 * kThinRows + c], top[3 * kThinRows + c])) * scale_log2 - kOffsetBelowMax<E>;
      if (mx > m[c] + kRescaleThreshold) {
        const float alpha = ex2(m[c] - mx);
        l[c] *= alpha;
        if (o_live) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
        m[c] = mx;
      }
    });
    if (o_live) {
      tmem_st16(o_tmem, o);
      tmem_wait_st();
    }
  }
  // P^T as the second operand: row c of 64 keys is 128 bytes, in the 128-byte swizzle
  uint8_t* dst = group.thin + (r >> 6) * kThinPanel + (r & 7) * 2;
  const int chunk = (r >> 3) & 7;
  thin_columns(cols, [&](int c) {
    if (!(c & 1)) {                                      // two columns at a time
      const float p0 = ex2(fmaf(__uint_as_float(sr[c]), scale_log2, -m[c])), p1 = ex2(fmaf(__uint_as_float(sr[c + 1]), scale_log2, -m[c + 1]));
      l[c] += p0;
      l[c + 1] += p1;
      const uint32_t w = pack2<E>(p0, p1);
      *reinterpret_cast<uint16_t*>(dst + c * 128 + ((chunk ^ (c & 7)) << 4)) = static_cast<uint16_t>(w);
      *reinterpret_cast<uint16_t*>(dst + (c + 1) * 128 + ((chunk ^ ((c + 1) & 7)) << 4)) = static_cast<uint16_t>(w >> 16);
    }
  });
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  mbar_arrive(bar_p_lo);
  mbar_arrive(bar_p_hi);
  return true;
}

// A unit of few rows: this thread is a key of each tile, and a channel of O^T.  Arrives on `over` where it has keys.  Returns the exchange's turns so far, or -1.
template <class E, int kD>
__device__ __noinline__ int thin_unit(const PagedKernelParams& p, const Seg s, PagedBarriers<kD>* bars, uint8_t* thin, uint32_t tmem_base, int count,
                                      int turns, uint64_t* over) {
  const int r = threadIdx.x & (kBlockM - 1), warp = r >> 5, lane = r & 31;
  const uint32_t s_tmem = tmem_base + (static_cast<uint32_t>(warp * 32) << 16), o_tmem = s_tmem + 2 * kBlockN;
  const AbortCtx ctx{&bars->abort_flag, p.status};
  ThinGroup group = {&bars->vote, thin, turns};
  const int cols = s.ntok * p.G;
  float m[kThinRows], l[kThinRows];
#pragma unroll
  for (int c = 0; c < kThinRows; ++c) {
    m[c] = kLowestOffset;
    l[c] = 0.f;
  }
  for (int j = 0; j < s.n_tiles; ++j) {
    if (!warp_wait(&bars->s_full[0], count & 1, ctx, SITE_PG_S)) return -1;
    tc_fence_after();
    ++count;
    const int key = (s.tile_begin + j) * kBlockN + r;
    int lo = 0, hi = key < s.len ? cols : 0;
    if (p.plan.causal && hi > 0) {
      const int64_t at = static_cast<int64_t>(key) - s.pos0, n = s.ntok;    // the first token that sees this key
      lo = static_cast<int>(min(max(at, static_cast<int64_t>(0)), n)) * p.G;
      if (p.plan.window > 0) hi = static_cast<int>(min(max(at + p.plan.window, static_cast<int64_t>(0)), n)) * p.G;
    }
    const auto wait_pv = [&]() {                           // of the tile before
      if (j == 0) return true;
      const bool done = warp_wait(&bars->pv_done[0], (count - 2) & 1, ctx, SITE_PG_O);
      tc_fence_after();
      return done;
    };
    if (!thin_softmax_tile<E>(s_tmem, o_tmem, group, ctx, p.scale_log2, cols, lo, hi, j > 0, m, l, smem_u32(&bars->s_free),
                              smem_u32(&bars->p_lo[0]), smem_u32(&bars->p_hi[0]), wait_pv))
      return -1;
  }
  uint32_t x[kThinRows];
  const float* sums = group.sums();
  if (s.n_tiles > 0) {
    if (!warp_wait(&bars->pv_done[0], (count - 1) & 1, ctx, SITE_PG_O)) return -1;
    tc_fence_after();
    tmem_ld16_sync(o_tmem, x);
    float mine = 0.f;
    thin_columns(cols, [&](int c) {
      float y = l[c];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (lane == c) mine = y;
    });
    if (lane < kThinRows) group.sums()[(warp & 3) * kThinRows + lane] = mine;
    if (!group.sync(ctx)) return -1;
  }
  thin_columns(cols, [&](int c) {
    if (c >= cols) return;
    float sum = 0.f, o = 0.f;
    if (s.n_tiles > 0) {
      sum = (sums[c] + sums[kThinRows + c]) + (sums[2 * kThinRows + c] + sums[3 * kThinRows + c]);
      o = __uint_as_float(x[c]);
    }
    if (s.slot >= 0) {
      float* slot = p.slots + s.slot * kSlotFloats<kD>;
      if (r < kD) slot[c * kD + r] = o;
      if (r == c) {
        slot[static_cast<size_t>(kSlotRows) * kD + c] = m[c];
        slot[static_cast<size_t>(kSlotRows) * (kD + 1) + c] = sum;
      }
    } else {
      const int i = c / p.G, h = s.hk * p.G + c - i * p.G;
      const float inv = sum != 0.f ? 1.0f / sum : 0.f;
      if (r < kD) {
        const uint32_t y = pack2<E>(o * inv, 0.f);
        reinterpret_cast<uint16_t*>(static_cast<E*>(p.o) + (s.tok0 + i) * p.o_stride_t + h * p.o_stride_h)[r] = static_cast<uint16_t>(y);
      }
      if (r == c && p.lse != nullptr) p.lse[static_cast<int64_t>(s.tok0 + i) * p.Hq + h] = sum != 0.f ? m[c] + log2f(sum) : -INFINITY;
    }
  });
  if (s.n_tiles > 0) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the second query tile may be copied here next
    tc_fence_before();
    mbar_arrive(smem_u32(over));
  }
  return group.turns;
}

// kThin: units of few rows are computed with keys as rows.  The 128 logits of a row leave no registers for that code beside
// them, in line or called: a chunk of 2048 tokens over 61234 keys takes 2710 us in the kernel that has it and 1970 us in the
// one that has not, 48 single tokens over 2000-32768 keys 340 and 425.  The launch takes the one that suits the mean number of
// rows a sequence brings.
template <class E, int kD, bool kThin>
__global__ void __launch_bounds__(kPagedThreads, 1) paged_attn_kernel(const __grid_constant__ PagedKernelParams p) {
  constexpr uint32_t kPanels = kD / 64;
  constexpr uint32_t kTile = kPanels * kPanelBytes;        // bytes of a 128-row tile
  using Bars = PagedBarriers<kD>;
  constexpr int kSlots = Bars::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem;
  {
    const uint32_t a = smem_u32(smem_raw);
    smem = smem_raw + (((a + 1023u) & ~1023u) - a);
  }
  uint8_t* smem_q = smem;
  uint8_t* smem_kv = smem + 2 * kTile;
  Bars* bars = reinterpret_cast<Bars*>(smem_kv + kRingBytes);
  PlanScratch* scratch = reinterpret_cast<PlanScratch*>(smem_kv);
  static_assert(sizeof(PlanScratch) <= kRingBytes, "the plan's scratch is the ring's memory");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int me = blockIdx.x, blocks = gridDim.x;
  AbortCtx ctx{&bars->abort_flag, p.status};
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (threadIdx.x == kMmaWarp * 32) {
    bars->abort_flag = 0;
    mbar_init(smem_u32(&bars->q_full), 1);
    mbar_init(smem_u32(&bars->q_empty), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars->s_full[i]), 1);
      mbar_init(smem_u32(&bars->p_lo[i]), kBlockM);
      mbar_init(smem_u32(&bars->p_hi[i]), kBlockM);
      mbar_init(smem_u32(&bars->pv_done[i]), 1);
      for (int k = 0; k < 2; ++k) mbar_init(smem_u32(&bars->o_free[i][k]), kBlockM);
    }
    mbar_init(smem_u32(&bars->s_free), kBlockM);
    mbar_init(smem_u32(&bars->vote), 4);
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(smem_u32(&bars->seg_full[i]), 1);
      mbar_init(smem_u32(&bars->seg_empty[i]), kSegReaders);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&bars->kv_full[i]), 1);
      mbar_init(smem_u32(&bars->kv_empty[i]), 1);
    }
    mbar_fence_init();
  }
  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&p.tmap_q);
    tma_prefetch_desc(&p.tmap_k);
    tma_prefetch_desc(&p.tmap_v);
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  // ------------------------------------------------------------------ the units of this block
  const BlockPlan bp = make_plan(p.plan, scratch, blocks, me);
  const int total = bp.rounds + bp.n_units;
  if (threadIdx.x == 0 && !bp.opens()) p.merge[me].pieces = 0;
  if (const int pieces = first_units(p.plan, scratch, bp, blocks, me, bars->units, bars->segs, kSegs)) {
    const Seg& s = bars->units.last;
    p.merge[me] = {pieces, s.tok0, s.ntok, s.hk};
  }
  // The plan's scratch was written with ordinary stores; the copies into the same memory go through the other proxy.
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  if (total == 0) {
    if (warp == 0) tmem_dealloc(tmem_base, kTmemCols);
    return;
  }
  const uint32_t g_magic = (65536u + p.G - 1) / p.G;       // r / G for r < 256 (G <= 128)

  // Unit i of this block, for each warp that takes them.
  bool ok = true;
  auto take = [&](int i) {
    if (i >= kSegs) ok = warp_wait(&bars->seg_full[i % kSegs], (i / kSegs - 1) & 1, ctx, SITE_PG_SEG);
    const Seg s = bars->segs[i % kSegs];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bars->seg_empty[i % kSegs]));
    return s;
  };

  if (warp == kLoadWarp) {
    // ---------------------------------------------------------------- TMA producer
    setmaxnreg_dec<kRegsService>();
    int n_q = 0, n_kv = 0;                                 // query blocks and places of the ring so far
    const int box = min(p.page_size, kBlockN);           // keys of a box
    const int boxes = kBlockN / box;
    const int per_page = max(p.page_size / kBlockN, 1);  // tiles of a page
    const int c = lane % boxes, panel = lane / boxes;
    const bool issues = panel < static_cast<int>(kPanels);
    bool thin_before = false;
    for (int si = 0; si < total && ok; ++si) {
      const Seg s = take(si);
      if (s.n_tiles == 0 || !ok) continue;
      const bool two = s.ntok > p.tile_tokens;
      if (n_q > 0) ok = warp_wait(&bars->q_empty, (n_q - 1) & 1, ctx, SITE_PG_QE);
      // A unit of few rows has its P in the second query tile's memory until its end: the unit before has to be over.
      if (ok && two && thin_before) {
        ok = warp_wait(o_free_of(bars, 0, n_q - 1), o_free_parity(n_q - 1), ctx, SITE_PG_QE);
        thin_before = false;
      }
      if (!ok) break;
      thin_before |= kThin && s.ntok * p.G <= kThinRows;
      if (lane == 0) {
        const uint32_t bar = smem_u32(&bars->q_full);
        mbar_expect_tx(bar, (two ? 2u : 1u) * kPanels * p.tile_tokens * p.G * 128u);
        for (int t = 0; t < (two ? 2 : 1); ++t)
          for (int pn = 0; pn < static_cast<int>(kPanels); ++pn)
            tma_load_4d(smem_u32(smem_q + t * kTile + pn * kPanelBytes), &p.tmap_q, bar, pn * 64, 0, s.tok0 + t * p.tile_tokens, s.hk);
      }
      ++n_q;
      // keys that some row of the block sees
      const int lo = keys_of(p.plan, s, 0).x, hi = keys_of(p.plan, s, s.ntok - 1).y;
      const int32_t* table = p.page_table + s.b * p.table_stride;
      const int none = max(p.pages, 1);                  // past the end: read as zeros
      // Looked at only where it is used, a tile or two later: a look at once would wait for memory with every tile.
      auto page_of = [&](int j) {
        const int tile = s.tile_begin + j, key = tile * kBlockN + c * box;
        return j >= s.n_tiles || key >= hi || key + box <= lo ? -1 : __ldg(table + (boxes > 1 ? tile * boxes + c : tile / per_page));
      };
      auto load = [&](bool is_v, int j, int page) {
        const int slot = n_kv % kSlots, use = n_kv / kSlots;
        if (use > 0) ok = warp_wait(&bars->kv_empty[slot], (use - 1) & 1, ctx, SITE_PG_KVE);
        if (!ok) return;
        const uint32_t bar = smem_u32(&bars->kv_full[slot]);
        if (lane == 0) mbar_expect_tx(bar, kTile);
        __syncwarp();
        const int row = boxes > 1 ? 0 : ((s.tile_begin + j) % per_page) * kBlockN;
        if (issues)
          tma_load_4d(smem_u32(smem_kv + slot * kTile + panel * kPanelBytes + c * box * 128), is_v ? &p.tmap_v : &p.tmap_k, bar,
                      panel * 64, row, s.hk, page < 0 || page >= p.pages ? none : page);
        ++n_kv;
      };
      int page = page_of(0), next = page_of(1);
      load(false, 0, page);
      for (int j = 0; j < s.n_tiles && ok; ++j) {
        const int after = page_of(j + 2);
        if (j + 1 < s.n_tiles) load(false, j + 1, next);
        if (ok) load(true, j, page);
        page = next;
        next = after;
      }
    }
    // The last uses of the ring and of Q end here, not in a block that has their memory next.
    for (int i = max(n_kv - kSlots, 0); i < n_kv && ok; ++i) ok = warp_wait(&bars->kv_empty[i % kSlots], (i / kSlots) & 1, ctx, SITE_PG_END);
    if (n_q > 0 && ok) ok = warp_wait(&bars->q_empty, (n_q - 1) & 1, ctx, SITE_PG_END);
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- issuer of S_t(j) = Q_t K_j^T
    setmaxnreg_dec<kRegsService>();
    const uint64_t q_desc = make_smem_desc_sw128(smem_u32(smem_q), 16, 1024);
    const uint64_t k_desc = make_smem_desc_sw128(smem_u32(smem_kv), 16, 1024);
    int n_q = 0, n_kv = 0, n_s = 0;                        // query blocks, places of the ring and S tiles so far
    for (int si = 0; si < total && ok; ++si) {
      const Seg s = take(si);
      const int n = s.n_tiles;
      if (n == 0 || !ok) continue;
      const int tiles = s.ntok > p.tile_tokens ? 2 : 1;
      const bool thin = kThin && s.ntok * p.G <= kThinRows;
      const uint32_t idesc = thin ? paged_idesc<E>(kThinRows, false) : paged_idesc<E>(kBlockN, false);
      ok = warp_wait(&bars->q_full, n_q & 1, ctx, SITE_PG_Q);
      ++n_q;
      for (int j = 0; j < n && ok; ++j) {
        const int place = n_kv + (j == 0 ? 0 : 2 * j - 1), slot = place % kSlots;
        ok = warp_wait(&bars->kv_full[slot], (place / kSlots) & 1, ctx, SITE_PG_KV);
        for (int t = 0; t < tiles && ok; ++t) {
          if (n_s > 0) ok = warp_wait(&bars->s_free, (n_s - 1) & 1, ctx, SITE_PG_SF);
          if (!ok) break;
          ++n_s;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t q0 = q_desc + ((t * kTile) >> 4), k0 = k_desc + ((slot * kTile) >> 4);
            const uint64_t a0 = thin ? k0 : q0, b0 = thin ? q0 : k0;
#pragma unroll
            for (int kk = 0; kk < kD / 16; ++kk) {
              const uint64_t off = static_cast<uint64_t>(((kk & 3) * 32 + (kk >> 2) * kPanelBytes) >> 4);
              mma_ss(tmem_base, a0 + off, b0 + off, idesc, kk > 0 ? 1u : 0u);
            }
            mma_commit(smem_u32(&bars->s_full[t]));
            if (t == tiles - 1) {
              mma_commit(smem_u32(&bars->kv_empty[slot]));
              if (j == n - 1) mma_commit(smem_u32(&bars->q_empty));
            }
          }
          __syncwarp();
        }
      }
      n_kv += 2 * n;
    }
  } else if (warp == kPvWarp) {
    // ---------------------------------------------------------------- issuer of O_t += P_t(j) V_j
    setmaxnreg_dec<kRegsService>();
    constexpr uint32_t idesc = paged_idesc<E>(kD, true);
    // V^T as the first operand is 128 rows: heads of 64 channels are read twice, into rows that nobody looks at
    constexpr uint32_t thin_idesc = paged_idesc<E>(kThinRows, false) | (1u << 15);
    const uint64_t vt_desc = make_smem_desc_sw128(smem_u32(smem_kv), kD == 128 ? kPanelBytes : 0, 1024);
    const uint64_t pt_desc = make_smem_desc_sw128(smem_u32(smem_q + kTile), 16, 1024);
    const uint64_t v_desc = make_smem_desc_sw128(smem_u32(smem_kv), kPanelBytes, 1024);
    int n_kv = 0, n_p[2] = {0, 0}, n_o[2] = {0, 0};        // places of the ring; P tiles and units of each group so far
    for (int si = 0; si < total && ok; ++si) {
      const Seg s = take(si);
      const int n = s.n_tiles;
      if (n == 0 || !ok) continue;
      const int tiles = s.ntok > p.tile_tokens ? 2 : 1;
      const bool thin = kThin && s.ntok * p.G <= kThinRows;
      const int lo = keys_of(p.plan, s, 0).x, hi = keys_of(p.plan, s, s.ntok - 1).y;
      for (int j = 0; j < n && ok; ++j) {
        const int place = n_kv + (j == n - 1 ? 2 * n - 1 : 2 * j + 2), slot = place % kSlots;
        ok = warp_wait(&bars->kv_full[slot], (place / kSlots) & 1, ctx, SITE_PG_KV);
        if (!ok) break;
        const int key0 = (s.tile_begin + j) * kBlockN;
        if (key0 < lo || key0 + kBlockN > hi) {
          // rows of V that nothing sees: a quarter of the warp a row, 16 bytes a lane
          const int from = max(lo - key0, 0), to = min(hi - key0, kBlockN);
          uint8_t* v = smem_kv + slot * kTile + (lane & 7) * 16;
          for (int i = lane >> 3; i < from + kBlockN - to; i += 4) {
            const int r = i < from ? i : to + i - from;
            for (uint32_t pn = 0; pn < kPanels; ++pn) *reinterpret_cast<uint4*>(v + pn * kPanelBytes + r * 128) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (t >= tiles || !ok) continue;
          const uint32_t parity = n_p[t] & 1;
          ++n_p[t];
          if (j == 0) {
            if (n_o[t] > 0) ok = warp_wait(o_free_of(bars, t, n_o[t] - 1), o_free_parity(n_o[t] - 1), ctx, SITE_PG_OF);
            ++n_o[t];
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (ok) ok = warp_wait(half == 0 ? &bars->p_lo[t] : &bars->p_hi[t], parity, ctx, half == 0 ? SITE_PG_P : SITE_PG_PH);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint64_t b0 = v_desc + ((slot * kTile) >> 4);
              const uint32_t d_tmem = tmem_base + (2 + t) * kBlockN, a_tmem = tmem_base + kBlockN + t * (kBlockN / 2);
              if (thin) {
                const uint64_t vt0 = vt_desc + ((slot * kTile) >> 4);
#pragma unroll
                for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                  mma_ss(d_tmem, vt0 + ((kk * 16 * 128) >> 4), pt_desc + (((kk & 3) * 32 + half * kThinPanel) >> 4), thin_idesc, (j > 0 || kk > 0) ? 1u : 0u);
              } else {
#pragma unroll
                for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                  mma_ts(d_tmem, a_tmem + kk * 8, b0 + ((kk * 16 * 128) >> 4), idesc, (j > 0 || kk > 0) ? 1u : 0u);
              }
              if (half == 1) {
                mma_commit(smem_u32(&bars->pv_done[t]));
                if (t == tiles - 1) mma_commit(smem_u32(&bars->kv_empty[slot]));
              }
            }
            __syncwarp();
          }
        }
      }
      n_kv += 2 * n;
    }
  } else if (warp < kMmaWarp) {
    // ---------------------------------------------------------------- softmax groups
    setmaxnreg_inc<kRegsSoftmax>();
    const int t = warp >> 2;
    const int r = threadIdx.x & (kBlockM - 1);           // row of the tile
    const int tok = div_small(r, g_magic), g = r - tok * p.G;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem_base + lane_off;
    const uint32_t p_tmem = s_tmem + kBlockN + t * (kBlockN / 2);
    const uint32_t o_tmem = s_tmem + (2 + t) * kBlockN;
    const uint32_t bar_s_free = smem_u32(&bars->s_free), bar_p_lo = smem_u32(&bars->p_lo[t]), bar_p_hi = smem_u32(&bars->p_hi[t]);
    int count = 0, n_o = 0;                              // tiles, and units with keys, of this group so far
    int turns = 0;                                       // of thin_unit's exchanges
    for (int si = 0; si < total && ok; ++si) {
      const Seg s = take(si);
      const int tokens = min(s.ntok - t * p.tile_tokens, p.tile_tokens);   // of this group's tile
      if (tokens <= 0 || !ok) continue;
      const bool live = tok < tokens;                    // a row that exists
      const bool works = (warp & 3) * 32 < tokens * p.G; // a warp that has any
      const int i = t * p.tile_tokens + tok;             // token of the block
      const int2 keys = live ? keys_of(p.plan, s, i) : make_int2(0, 0);
      // within [all_lo, all_hi) no row of the tile needs a mask
      const int all_hi = keys_of(p.plan, s, t * p.tile_tokens).y, all_lo = keys_of(p.plan, s, t * p.tile_tokens + tokens - 1).x;
      if (kThin && s.ntok * p.G <= kThinRows) {
        turns = thin_unit<E, kD>(p, s, bars, smem_q + kTile, tmem_base, count, turns, o_free_of(bars, 0, n_o));
        ok = turns >= 0;
        count += s.n_tiles;
        n_o += s.n_tiles > 0;
        continue;
      }
      float m_used = kLowestOffset, l_sum = 0.f;
      for (int j = 0; j < s.n_tiles && ok; ++j) {
        ok = warp_wait(&bars->s_full[t], count & 1, ctx, SITE_PG_S);
        if (!ok) break;
        tc_fence_after();
        ++count;
        auto wait_pv = [&]() {
          if (j == 0) return true;
          const bool done = warp_wait(&bars->pv_done[t], (count - 2) & 1, ctx, SITE_PG_O);
          tc_fence_after();
          return done;
        };
        const int key0 = (s.tile_begin + j) * kBlockN;
        if (works) {
          ok = paged_softmax_tile<E, kD>(s_tmem, p_tmem, o_tmem, p.scale_log2, key0 < all_lo || key0 + kBlockN > all_hi, keys.x - key0,
                                         keys.y - key0, j > 0, m_used, l_sum, bar_s_free, bar_p_lo, bar_p_hi, wait_pv);
        } else {
          // no row: S is left unread and P as it is, a tile's turn all the same
          tc_fence_before();
          mbar_arrive(bar_s_free);
          ok = wait_pv();
          mbar_arrive(bar_p_lo);
          mbar_arrive(bar_p_hi);
        }
      }
      if (!ok) break;
      if (s.n_tiles > 0) {
        ok = warp_wait(&bars->pv_done[t], (count - 1) & 1, ctx, SITE_PG_O);
        if (!ok) break;
        tc_fence_after();
      }
      if (works) {
        const int row = t * kBlockM + r;
        if (s.slot >= 0) {
          float* slot = p.slots + s.slot * kSlotFloats<kD>;
          float4* dst = reinterpret_cast<float4*>(slot + static_cast<size_t>(row) * kD);
          if (s.n_tiles > 0) {
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) {
              uint32_t x[32];
              tmem_ld32_sync(o_tmem + c * 32, x);
              if (live) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  dst[c * 8 + k] = make_float4(__uint_as_float(x[4 * k]), __uint_as_float(x[4 * k + 1]), __uint_as_float(x[4 * k + 2]),
                                               __uint_as_float(x[4 * k + 3]));
              }
            }
          }
          if (live) {
            slot[static_cast<size_t>(kSlotRows) * kD + row] = m_used;
            slot[static_cast<size_t>(kSlotRows) * (kD + 1) + row] = l_sum;
          }
        } else {
          const float inv = l_sum != 0.f ? 1.0f / l_sum : 0.f;
          const int h = s.hk * p.G + g;
          E* dst = static_cast<E*>(p.o) + (s.tok0 + i) * p.o_stride_t + h * p.o_stride_h;
#pragma unroll
          for (int c = 0; c < kD / 32; ++c) {
            uint32_t x[32];
            if (s.n_tiles > 0) {
              tmem_ld32_sync(o_tmem + c * 32, x);
            } else {
#pragma unroll
              for (int k = 0; k < 32; ++k) x[k] = 0u;
            }
            if (live) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t y[4];
#pragma unroll
                for (int v = 0; v < 4; ++v)
                  y[v] = pack2<E>(__uint_as_float(x[8 * k + 2 * v]) * inv, __uint_as_float(x[8 * k + 2 * v + 1]) * inv);
                reinterpret_cast<uint4*>(dst)[c * 4 + k] = make_uint4(y[0], y[1], y[2], y[3]);
              }
            }
          }
          if (live && p.lse != nullptr)
            p.lse[static_cast<int64_t>(s.tok0 + i) * p.Hq + h] = l_sum != 0.f ? m_used + log2f(l_sum) : -INFINITY;
        }
      }
      if (s.n_tiles > 0) {
        tc_fence_before();
        mbar_arrive(smem_u32(o_free_of(bars, t, n_o++)));
      }
    }
  } else {
    // ---------------------------------------------------------------- the other units of this block
    setmaxnreg_dec<kRegsService>();
    if (lane == 0 && total > kSegs) {
      for (UnitWalk w(p.plan, bars->units, bp.rounds, total, kSegs); w.more(); w.next(p.plan)) {
        ok = mbar_wait(smem_u32(&bars->seg_empty[w.i % kSegs]), (w.i / kSegs - 1) & 1, ctx, SITE_PG_SEGE);
        if (!ok) break;
        bars->segs[w.i % kSegs] = w.seg(p.plan, bars->units);
        mbar_arrive(smem_u32(&bars->seg_full[w.i % kSegs]));
      }
    }
    __syncwarp();
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  if (__syncthreads_or(!ok)) {
    // Give copies and MMAs that are still in flight time to land before the memory they target is released.
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc(tmem_base, kTmemCols);
}

// States of a unit's pieces -> its rows.  Block (k, y) merges rows y, y + gridDim.y, ... of the unit whose first piece block k
// of the attention kernel swept: piece 0 is that block's slot 2 k + 1, piece i > 0 slot 2 (k + i).  A warp a row, its lanes
// looking up a piece each and then reading four pieces' rows at a time; few rows of many pieces (a long sequence of few rows
// over the whole chip): the warps share a row's pieces.
constexpr int kMergeWarps = 8;

template <class E, int kD>
__global__ void __launch_bounds__(32 * kMergeWarps) paged_merge_kernel(const float* __restrict__ slots, const MergeDesc* __restrict__ descs, E* o,
                                                                      int64_t o_stride_t, int64_t o_stride_h, float* lse, int Hq, int G,
                                                                      int tile_tokens) {
  constexpr int kPer = kD / 32;                            // channels a lane
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const MergeDesc d = descs[blockIdx.x];
  if (d.pieces < 2) return;
  __shared__ float part[kMergeWarps][kD + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows0 = min(d.ntok, tile_tokens) * G, rows = d.ntok * G;
  const bool shared = d.pieces > 4 && rows <= 2 * static_cast<int>(gridDim.y);
  const int step = shared ? 1 : kMergeWarps;
  for (int base = blockIdx.y * step; base < rows; base += gridDim.y * step) {
    const int x = shared ? base : base + warp;             // row of the unit
    if (x >= rows) continue;                               // whole warps, and only where no barrier follows
    const int row = x < rows0 ? x : kBlockM + x - rows0;   // of its slots
    const int first = shared ? warp : 0, by = shared ? kMergeWarps : 1;
    float m = kLowestOffset, l = 0.f, acc[kPer];
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] = 0.f;
    auto slot_of = [&](int i) { return slots + static_cast<size_t>(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * kSlotFloats<kD>; };
    for (int i0 = first; i0 < d.pieces; i0 += 32 * by) {
      const int mine = i0 + lane * by, n = min((d.pieces - i0 + by - 1) / by, 32);
      float li = 0.f, mi = 0.f;
      if (mine < d.pieces) {
        const float* s = slot_of(mine);
        li = s[static_cast<size_t>(kSlotRows) * (kD + 1) + row];
        mi = s[static_cast<size_t>(kSlotRows) * kD + row];
      }
      // A state is left out where its sum is 0, and only there: a NaN sum is the row's result.
      const uint32_t some = __ballot_sync(0xffffffffu, li != 0.f);
      float m_new = li != 0.f ? fmaxf(m, mi) : m;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, x));
      const float w_old = exp2f(m - m_new), w = li != 0.f ? exp2f(mi - m_new) : 0.f;
      float sum = li != 0.f ? li * w : 0.f;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      m = m_new;
      l = l * w_old + sum;
#pragma unroll
      for (int c = 0; c < kPer; ++c) acc[c] *= w_old;
      for (int k0 = 0; k0 < n; k0 += 4) {
        float v[4][kPer], wk[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          wk[k] = __shfl_sync(0xffffffffu, w, (k0 + k) & 31);
#pragma unroll
          for (int c = 0; c < kPer; ++c) v[k][c] = 0.f;
          if (k0 + k < n && (some >> (k0 + k) & 1)) {
            const float* src = slot_of(i0 + (k0 + k) * by) + static_cast<size_t>(row) * kD + lane * kPer;
            if (kPer == 4) *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(src);
            else *reinterpret_cast<float2*>(v[k]) = *reinterpret_cast<const float2*>(src);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k0 + k < n && (some >> (k0 + k) & 1)) {
#pragma unroll
            for (int c = 0; c < kPer; ++c) acc[c] += v[k][c] * wk[k];
          }
      }
    }
    if (shared) {
#pragma unroll
      for (int c = 0; c < kPer; ++c) part[warp][lane * kPer + c] = acc[c];
      if (lane == 0) { part[warp][kD] = m; part[warp][kD + 1] = l; }
      __syncthreads();
      if (warp == 0) {
        float top = kLowestOffset;
#pragma unroll
        for (int i = 0; i < kMergeWarps; ++i) top = fmaxf(top, part[i][kD]);
        l = 0.f;
#pragma unroll
        for (int c = 0; c < kPer; ++c) acc[c] = 0.f;
        for (int i = 0; i < kMergeWarps; ++i) {
          if (part[i][kD + 1] == 0.f) continue;
          const float w = exp2f(part[i][kD] - top);
          l += part[i][kD + 1] * w;
#pragma unroll
          for (int c = 0; c < kPer; ++c) acc[c] += part[i][lane * kPer + c] * w;
        }
        m = top;
      }
    }
    if (!shared || warp == 0) {
      const float inv = l != 0.f ? 1.0f / l : 0.f;
      const int tok = x / G, h = d.hk * G + x - tok * G;
      E* dst = o + (d.tok0 + tok) * o_stride_t + h * o_stride_h + lane * kPer;
      if (kPer == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<E>(acc[0] * inv, acc[1] * inv), pack2<E>(acc[kPer - 2] * inv, acc[kPer - 1] * inv));
      else *reinterpret_cast<uint32_t*>(dst) = pack2<E>(acc[0] * inv, acc[1] * inv);
      if (lse != nullptr && lane == 0) lse[static_cast<int64_t>(d.tok0 + tok) * Hq + h] = l != 0.f ? m + log2f(l) : -INFINITY;
    }
    if (shared) __syncthreads();
  }
}

}  // namespace dtb
