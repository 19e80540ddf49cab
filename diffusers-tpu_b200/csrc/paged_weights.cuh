// The attention that each key of a paged cache got from the new tokens, for sm_100a.
//
// Keys as rows.  S^T = K Q^T puts a key on each of the 128 rows of a tile, so a thread owns a key, adds up
// 2^(s - lse) over the columns - the query rows of attn (token, head of the group) - in a register, and no thread needs
// another's result; lse, one number a column, is read from shared memory as a broadcast.  The columns of a tile are rounded up
// to 16, so that a decode step of a few rows costs a few columns.
//
// A block takes an equal part of all items, an item being 512 keys of one key head: four tiles, one for each group of four
// warps.  (Two groups of four, each with two S tiles in turn, left the exponentials' unit idle for half the time: the 64 tokens
// x 24 heads of two prompts of 30000-60000 keys took 81 us, and no less with fewer instructions.)  K tiles come through a ring of 160 KB; up to two query tiles stay in shared memory for all items of a head,
// more are streamed for each.  A single token's step is bound by the keys' bytes, many tokens by the exponentials: 16 a
// cycle and SM.
#pragma once

#include "paged_attn.cuh"

namespace dtb {

constexpr int kGroups = 4;                   // key tiles of an item
constexpr int kItemKeys = kGroups * kBlockN;
constexpr int kWeightsThreads = (kGroups * 4 + 4) * 32;
constexpr int kWeightsMma = kGroups * 4, kWeightsLoad = kWeightsMma + 1, kWeightsFill = kWeightsMma + 2;   // warps behind the groups'
constexpr int kFillSlots = 4096;             // slots that the idle warp fills at a time

struct WeightsKernelParams {
  CUtensorMap tmap_q, tmap_k;
  PlanParams plan;                           // block_tokens: tokens of a query tile
  const int32_t* page_table;
  int64_t table_stride;
  int pages, page_size;
  const float* lse;
  const float* prior;
  float* out;
  int64_t prior_stride_b, prior_stride_h, out_stride_b, out_stride_h;
  int32_t* status;
  int Hq, G;
  float scale_log2;
};

struct WeightsScratch {
  int64_t weight[kPlanMaxSeqs + 1];
  int64_t warp_w[kWeightsThreads / 32];
};

template <int kD>
struct __align__(16) WeightsBarriers {
  static constexpr int kSlots = kRingBytes / (128 * kD * 2);
  float neg_lse[2][kBlockM];
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[kSlots], kv_empty[kSlots];
  uint64_t s_full[kGroups], s_free[kGroups];
  uint32_t tmem_base;
  int abort_flag;
};

template <int kD>
constexpr size_t kWeightsSmem = 1024 + 2 * 128 * kD * 2 + kRingBytes + sizeof(WeightsBarriers<kD>);
static_assert(kWeightsSmem<128> <= 232448, "more shared memory than a block can have");

enum WeightsSite : int { SITE_KW_Q = 210, SITE_KW_QE = 215, SITE_KW_K = 220, SITE_KW_KE = 230, SITE_KW_S = 240, SITE_KW_SF = 245, SITE_KW_END = 250 };

// Items of one sequence, and what each costs: its keys' bytes or the exponentials of its columns.
struct SeqItems {
  SeqPlan s;
  int rows;                // query rows of a head
  int first, n;            // items of a head: [first, first + n)
  int cost;
};

__device__ __forceinline__ SeqItems seq_items(const PlanParams& p, int G, int b) {
  SeqItems q;
  q.s = seq_plan(p, b);
  q.rows = q.s.n * G;
  // keys that no new token sees keep what they have
  const int64_t lowest = p.causal && p.window > 0 ? static_cast<int64_t>(q.s.pos0) - p.window + 1 : 0;
  q.first = static_cast<int>(min(max(lowest, static_cast<int64_t>(0)), static_cast<int64_t>(q.s.len)) / kItemKeys);
  q.n = q.s.n > 0 ? (q.s.len + kItemKeys - 1) / kItemKeys - q.first : 0;
  q.cost = max(180, min(q.rows, 1 << 20) + 20);
  return q;
}

template <class E, int kD>
__global__ void __launch_bounds__(kWeightsThreads, 1) key_weights_kernel(const __grid_constant__ WeightsKernelParams p) {
  constexpr uint32_t kPanels = kD / 64;
  constexpr uint32_t kTile = kPanels * kPanelBytes;
  using Bars = WeightsBarriers<kD>;
  constexpr int kSlots = Bars::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem;
  {
    const uint32_t a = smem_u32(smem_raw);
    smem = smem_raw + (((a + 1023u) & ~1023u) - a);
  }
  uint8_t* smem_q = smem;
  uint8_t* smem_k = smem + 2 * kTile;
  Bars* bars = reinterpret_cast<Bars*>(smem_k + kRingBytes);
  WeightsScratch* sc = reinterpret_cast<WeightsScratch*>(smem_k);
  static_assert(sizeof(WeightsScratch) <= kRingBytes, "the scratch is the ring's memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int me = blockIdx.x, blocks = gridDim.x;
  AbortCtx ctx{&bars->abort_flag, p.status};

  if (tid == kWeightsMma * 32) {
    bars->abort_flag = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars->q_full[i]), 2);                  // the copy, and lse
      mbar_init(smem_u32(&bars->q_empty[i]), 1 + kGroups * 4);   // the products, and the warps that read lse
    }
    for (int i = 0; i < kGroups; ++i) {
      mbar_init(smem_u32(&bars->s_full[i]), 1);
      mbar_init(smem_u32(&bars->s_free[i]), kBlockN);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&bars->kv_full[i]), 1);
      mbar_init(smem_u32(&bars->kv_empty[i]), 1);
    }
    mbar_fence_init();
  }
  if (warp == kWeightsLoad && lane == 0) {
    tma_prefetch_desc(&p.tmap_q);
    tma_prefetch_desc(&p.tmap_k);
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  // ------------------------------------------------------------------ this block's items: an equal part of their cost
  int64_t total = 0;
  for (int b0 = 0; b0 < p.plan.B; b0 += kWeightsThreads) {
    const int b = b0 + tid;
    int64_t w = 0;
    if (b < p.plan.B) {
      const SeqItems q = seq_items(p.plan, p.G, b);
      w = static_cast<int64_t>(q.n) * q.cost * p.plan.Hkv;
    }
    int64_t inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sc->warp_w[warp] = inc;
    __syncthreads();
    int64_t before = total;
#pragma unroll
    for (int i = 0; i < kWeightsThreads / 32; ++i) {
      if (i < warp) before += sc->warp_w[i];
      total += sc->warp_w[i];
    }
    if (b < p.plan.B) sc->weight[b] = before + inc - w;
    __syncthreads();
  }
  // first item that starts at or behind x: sequence, and its number among the sequence's
  auto item_at = [&](int64_t x) {
    if (x >= total) return make_int2(p.plan.B, 0);
    const int b = last_at_most(sc->weight, p.plan.B, x);
    const SeqItems q = seq_items(p.plan, p.G, b);
    const int64_t i = (x - sc->weight[b] + q.cost - 1) / q.cost;
    return make_int2(b, static_cast<int>(i));            // may be one past the sequence's last
  };
  const int64_t share = (total + blocks - 1) / blocks;
  const int2 from = item_at(min(share * me, total)), to = item_at(min(share * (me + 1), total));
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  bool ok = true;

  // The runs of this block: consecutive items of one key head.  f(q, b, hk, first item, number of items).
  auto for_runs = [&](auto f) {
    int b = from.x, at = from.y;
    while (ok && b < p.plan.B && b <= to.x) {
      const SeqItems q = seq_items(p.plan, p.G, b);
      const int end = b < to.x ? q.n * p.plan.Hkv : min(to.y, q.n * p.plan.Hkv);
      while (ok && at < end) {
        const int hk = at / q.n, i = at - hk * q.n, n = min(q.n - i, end - at);
        f(q, b, hk, q.first + i, n);
        at += n;
      }
      ++b;
      at = 0;
    }
  };
  const int tile_rows = p.plan.block_tokens * p.G;       // of a full query tile

  if (warp == kWeightsLoad) {
    // ---------------------------------------------------------------- TMA producer
    int n_k = 0, n_q = 0;
    const int box = min(p.page_size, kBlockN), boxes = kBlockN / box, per_page = max(p.page_size / kBlockN, 1);
    const int c = lane % boxes, panel = lane / boxes;
    for_runs([&](const SeqItems& q, int b, int hk, int first, int n) {
      const int q_tiles = (q.rows + tile_rows - 1) / tile_rows;
      auto load_q = [&](int t) {
        const int slot = n_q & 1, use = n_q >> 1;
        if (use > 0) ok = warp_wait(&bars->q_empty[slot], (use - 1) & 1, ctx, SITE_KW_QE);
        if (!ok) return;
        const uint32_t bar = smem_u32(&bars->q_full[slot]);
        const int tok0 = q.s.first + t * p.plan.block_tokens;
        if (lane == 0) {
          mbar_expect_tx(bar, kPanels * tile_rows * 128u);
          for (int pn = 0; pn < static_cast<int>(kPanels); ++pn)
            tma_load_4d(smem_u32(smem_q + slot * kTile + pn * kPanelBytes), &p.tmap_q, bar, pn * 64, 0, tok0, hk);
        }
        const int rows = min(q.rows - t * tile_rows, tile_rows);
        for (int r = lane; r < kBlockM; r += 32) {
          const int tok = r / p.G;
          bars->neg_lse[slot][r] = r < rows ? -p.lse[static_cast<int64_t>(tok0 + tok) * p.Hq + hk * p.G + r - tok * p.G] : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
        ++n_q;
      };
      const int32_t* table = p.page_table + b * p.table_stride;
      const int none = max(p.pages, 1);
      const int end = (q.s.len + kBlockN - 1) / kBlockN;                 // tiles of the sequence
      const int t0 = first * kGroups, t1 = min((first + n) * kGroups, end);
      // Looked at only where it is used, two tiles later: a look at once would wait for memory with every tile.
      auto page_of = [&](int tile) {
        return tile >= t1 || tile * kBlockN + c * box >= q.s.len ? -1 : __ldg(table + (boxes > 1 ? tile * boxes + c : tile / per_page));
      };
      int page = page_of(t0), next = page_of(t0 + 1);
      for (int tile = t0; tile < t1 && ok; ++tile) {
        const int after = page_of(tile + 2);
        const int slot = n_k % kSlots, use = n_k / kSlots;
        if (use > 0) ok = warp_wait(&bars->kv_empty[slot], (use - 1) & 1, ctx, SITE_KW_KE);
        if (!ok) break;
        const uint32_t bar = smem_u32(&bars->kv_full[slot]);
        if (lane == 0) mbar_expect_tx(bar, kTile);
        __syncwarp();
        if (panel < static_cast<int>(kPanels))
          tma_load_4d(smem_u32(smem_k + slot * kTile + panel * kPanelBytes + c * box * 128), &p.tmap_k, bar, panel * 64,
                      boxes > 1 ? 0 : (tile % per_page) * kBlockN, hk, page < 0 || page >= p.pages ? none : page);
        ++n_k;
        page = next;
        next = after;
        // the queries follow the item's keys: all of them once a run, or, more than fit, for each item
        if (tile % kGroups == kGroups - 1 || tile == t1 - 1) {
          if (q_tiles > 2 || tile < t0 + kGroups)
            for (int t = 0; t < q_tiles && ok; ++t) load_q(t);
        }
      }
    });
    for (int i = max(n_k - kSlots, 0); i < n_k && ok; ++i) ok = warp_wait(&bars->kv_empty[i % kSlots], (i / kSlots) & 1, ctx, SITE_KW_END);
    for (int i = max(n_q - 2, 0); i < n_q && ok; ++i) ok = warp_wait(&bars->q_empty[i & 1], (i >> 1) & 1, ctx, SITE_KW_END);
  } else if (warp == kWeightsMma) {
    // ---------------------------------------------------------------- issuer of S^T = K_g Q_t^T: one thread, no votes
    if (elect_one()) {
      int k_slot = 0, n_q = 0;                              // place of the ring that the item starts at; query tiles so far
      uint32_t k_use = 0, s_use = 0;                        // its uses before; parities of the groups' next turns
      const uint64_t q_desc = make_smem_desc_sw128(smem_u32(smem_q), 16, 1024), k_desc = make_smem_desc_sw128(smem_u32(smem_k), 16, 1024);
      for_runs([&](const SeqItems& q, int, int, int first, int n) {
        const int q_tiles = (q.rows + tile_rows - 1) / tile_rows;
        const bool stay = q_tiles <= 2;
        const int end = (q.s.len + kBlockN - 1) / kBlockN;
        for (int it = 0; it < n && ok; ++it) {
          const int groups = min(end - (first + it) * kGroups, kGroups);
          for (int t = 0; t < q_tiles && ok; ++t) {
            const int place = stay ? n_q + t : n_q;
            ok = mbar_wait(smem_u32(&bars->q_full[place & 1]), (place >> 1) & 1, ctx, SITE_KW_Q);
            const int cols = (min(q.rows - t * tile_rows, tile_rows) + 15) & ~15;
            const uint32_t idesc = paged_idesc<E>(16, false) + (static_cast<uint32_t>((cols - 16) >> 3) << 17);
            const uint64_t b0 = q_desc + (((place & 1) * kTile) >> 4);
            int ks = k_slot;
            uint32_t use = k_use;
            for (int g = 0; g < groups && ok; ++g) {
              if (t == 0) ok = mbar_wait(smem_u32(&bars->kv_full[ks]), use & 1, ctx, SITE_KW_K);
              // a bit a group: the parity of its last turn's end, once it has had one
              if (ok && (s_use >> (g + 8) & 1)) ok = mbar_wait(smem_u32(&bars->s_free[g]), (s_use >> g) & 1, ctx, SITE_KW_SF);
              if (!ok) break;
              s_use = (s_use >> (g + 8) & 1) ? s_use ^ (1u << g) : s_use | (1u << (g + 8));
              tc_fence_after();
              const uint64_t a0 = k_desc + ((ks * kTile) >> 4);
#pragma unroll
              for (int kk = 0; kk < kD / 16; ++kk) {
                const uint64_t off = static_cast<uint64_t>(((kk & 3) * 32 + (kk >> 2) * kPanelBytes) >> 4);
                mma_ss(tmem_base + g * kBlockM, a0 + off, b0 + off, idesc, kk > 0 ? 1u : 0u);
              }
              mma_commit(smem_u32(&bars->s_full[g]));
              if (t == q_tiles - 1) mma_commit(smem_u32(&bars->kv_empty[ks]));
              if (++ks == kSlots) { ks = 0; ++use; }
            }
            if (ok && (!stay || it == n - 1)) mma_commit(smem_u32(&bars->q_empty[place & 1]));
            if (!stay) ++n_q;
          }
          k_slot += groups;
          if (k_slot >= kSlots) { k_slot -= kSlots; ++k_use; }
        }
        if (stay) n_q += q_tiles;
      });
    }
    ok = __all_sync(0xffffffffu, ok);
  } else if (warp < kWeightsMma) {
    // ---------------------------------------------------------------- a thread per key
    const int g = warp >> 2, r = tid & (kBlockN - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
    int n_q = 0, n_s = 0;
    for_runs([&](const SeqItems& q, int b, int hk, int first, int n) {
      const int q_tiles = (q.rows + tile_rows - 1) / tile_rows;
      const bool stay = q_tiles <= 2;
      const int slots = static_cast<int>(p.plan.capacity);
      const float* prior = p.prior != nullptr ? p.prior + b * p.prior_stride_b + hk * p.prior_stride_h : nullptr;
      float* out = p.out + b * p.out_stride_b + hk * p.out_stride_h;
      const int before = q.s.pos0;                                       // slot of the first new token
      // What a key had is asked for an item ahead, in place: where the compiler puts an ordinary load, in front of its use, each
      // item waited for memory.
      auto ask = [&](int it) {
        const int key = (first + it) * kItemKeys + g * kBlockN + r;
        float x = 0.f;
        if (prior != nullptr && it < n && key < q.s.len) asm volatile("ld.global.f32 %0, [%1];" : "=f"(x) : "l"(prior + key) : "memory");
        return x;
      };
      float next = ask(0);
      for (int it = 0; it < n && ok; ++it) {
        const int key0 = (first + it) * kItemKeys + g * kBlockN, key = key0 + r;
        const bool there = key0 < q.s.len;                               // the item has this group's tile
        const float had = next;
        next = ask(it + 1);
        float sum = 0.f;
        // new tokens [first_tok, end_tok) see this key; far outside the new ones, any number does
        const int64_t at = static_cast<int64_t>(key) - before;
        const int first_tok = static_cast<int>(max(min(at, static_cast<int64_t>(1 << 30)), static_cast<int64_t>(-(1 << 30))));
        const int end_tok = static_cast<int>(max(min(at + p.plan.window, static_cast<int64_t>(1 << 30)), static_cast<int64_t>(-(1 << 30))));
        for (int t = 0; t < q_tiles && ok; ++t) {
          const int place = stay ? n_q + t : n_q;
          ok = warp_wait(&bars->q_full[place & 1], (place >> 1) & 1, ctx, SITE_KW_Q);
          if (ok && there) {
            ok = warp_wait(&bars->s_full[g], n_s & 1, ctx, SITE_KW_S);
            if (!ok) break;
            ++n_s;
            tc_fence_after();
            // columns of the tokens that see this key
            const int cols = min(q.rows - t * tile_rows, tile_rows);
            int lo = 0, hi = cols;
            if (p.plan.causal) {
              lo = min(min(max(first_tok - t * p.plan.block_tokens, 0), p.plan.block_tokens) * p.G, cols);
              if (p.plan.window > 0) hi = min(min(max(end_tok - t * p.plan.block_tokens, 0), p.plan.block_tokens) * p.G, cols);
            }
            const uint32_t s_tmem = tmem_base + lanes + g * kBlockM;
            const float4* lse = reinterpret_cast<const float4*>(bars->neg_lse[place & 1]);
            uint64_t acc[4] = {0, 0, 0, 0};
            // 16 of the columns in registers, from column c0 on, stage by stage.
            auto add_as = [&](auto masked, int c0, const uint32_t* s) {
              float x[16];
#pragma unroll
              for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(x + i) = lse[(c0 + i) >> 2];
#pragma unroll
              for (int i = 0; i < 16; i += 2)
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale2, pack_f32x2(x[i], x[i + 1])), x[i], x[i + 1]);
              if (decltype(masked)::value) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (c0 + i < lo || c0 + i >= hi) x[i] = -INFINITY;
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = ex2(x[i]);
#pragma unroll
              for (int i = 0; i < 16; i += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = add_f32x2(acc[k], pack_f32x2(x[i + 2 * k], x[i + 2 * k + 1]));
            };
            auto add = [&](int c0, const uint32_t* s) {
              if (__any_sync(0xffffffffu, c0 < lo || c0 + 16 > hi)) add_as(std::true_type(), c0, s);
              else add_as(std::false_type(), c0, s);
            };
            const uint32_t s_free = smem_u32(&bars->s_free[g]);
            if (cols <= 16) {
              uint32_t s[16];
              tmem_ld16_sync(s_tmem, s);
              tc_fence_before();
              mbar_arrive(s_free);
              add(0, s);
            } else {
              // columns behind the last are whatever was there, and masked
              for (int c1 = 0; c1 < cols; c1 += 32) {
                uint32_t s[32];
                tmem_ld32_sync(s_tmem + c1, s);
                if (c1 + 32 >= cols) {
                  tc_fence_before();
                  mbar_arrive(s_free);
                }
                add(c1, s);
                if (c1 + 16 < cols) add(c1 + 16, s + 16);
              }
            }
            float a0, a1;
            unpack_f32x2(add_f32x2(add_f32x2(acc[0], acc[1]), add_f32x2(acc[2], acc[3])), a0, a1);
            sum += a0 + a1;
          }
          if (!stay || it == n - 1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->q_empty[place & 1]));
          }
          if (!stay) ++n_q;
        }
        if (ok && key < slots) out[key] = key < q.s.len ? had + sum : 0.f;
      }
      if (stay) n_q += q_tiles;
    });
  } else if (warp == kWeightsFill) {
    // ---------------------------------------------------------------- slots that no item has: what they had, and zeros
    const int64_t slots = p.plan.capacity, parts = (slots + kFillSlots - 1) / kFillSlots;
    const int64_t work = parts * p.plan.B * p.plan.Hkv;
    for (int64_t w = me; w < work; w += blocks) {
      const int64_t row = w / parts;
      const int b = static_cast<int>(row / p.plan.Hkv), hk = static_cast<int>(row % p.plan.Hkv);
      const SeqItems q = seq_items(p.plan, p.G, b);
      const int64_t begin = (w - row * parts) * kFillSlots, end = min(begin + kFillSlots, slots);
      const int64_t i0 = static_cast<int64_t>(q.first) * kItemKeys, i1 = i0 + static_cast<int64_t>(q.n) * kItemKeys;   // slots of items
      float* out = p.out + b * p.out_stride_b + hk * p.out_stride_h;
      const float* prior = p.prior != nullptr ? p.prior + b * p.prior_stride_b + hk * p.prior_stride_h : nullptr;
      for (int64_t i = begin + lane; i < end; i += 32) {
        if (i >= i0 && i < i1) continue;
        out[i] = prior != nullptr && i < q.s.len ? prior[i] : 0.f;
      }
    }
  }
  tc_fence_before();
  if (__syncthreads_or(!ok)) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc(tmem_base, kTmemCols);
}

}  // namespace dtb
