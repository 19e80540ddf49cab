// Who does what in a launch over ragged sequences whose lengths only the device knows.
//
// Work is counted in units: one query block (up to kTokens new tokens times the query heads of a group) of one key head of one
// sequence.  A unit weighs the keys that it sees plus kUnitCost for its start and finish, times what a key of it costs beside
// those of other units, and all units lie end to end in the order (sequence, head, query block), so that a place on that line is a unit and a key of it.  Every block of a launch
// computes the same plan from query_start and kv_len and takes its own part, so that a captured launch follows the lengths
// it finds, and no block waits for another:
//   * the line is cut into as many equal ranges as there are blocks, each swept by one block.  Units that a cut goes through
//     are swept in pieces, whose states a second kernel merges; a cut close to an end of its unit moves there.
//   * where several query blocks sweep the same long keys, whole units are dealt out first, in rounds of one a block: blocks
//     of a round start at the same key together, and what one reads the others find in L2.  Only the units behind the last
//     full round are cut, and each block's range of them makes up for what it was dealt.
#pragma once

#include "paged.cuh"

namespace dtb {

constexpr int kPlanThreads = 384;
constexpr int kPlanTile = 128;             // keys of a tile
// Keys that a unit's start and finish cost as much time as; also the shortest range, so that a block takes no second unit
// while others have none.
constexpr int kUnitCost = 384;
// A cut leaves at least so many keys on both sides of itself.
constexpr int kLeastKeys = 512;
// Mean cost, in cheap keys, from which units that share keys are dealt out whole.  (From twice as many: 2048 tokens x 40 heads
// over 5000 keys 201 us for 178, 4 x 5000 tokens x 24 heads 723 for 721; from half as many 177 and 743.)
constexpr int kLongUnit = 4096;
// A key's cost is counted in eighths of a cheap one's.
constexpr int kKeyCost = 8;
constexpr int kPlanMaxBlocks = 160;
constexpr int kPlanMaxRounds = 64;
constexpr int kPlanMaxSeqs = 8192;

struct PlanParams {
  const int32_t* query_start;
  const int32_t* kv_len;
  int64_t capacity;        // slots that a row of the page table can name
  int B, T, Hkv;
  int block_tokens;        // new tokens of a query block
  int causal, window;
  // What a key of a sequence's units costs: kKeyCost for up to cheap_tokens new tokens, cost_one up to tile_tokens, else cost_two.
  int cheap_tokens = 0, tile_tokens = 0, cost_one = kKeyCost, cost_two = kKeyCost;
};

// What the plan needs of one sequence.
struct SeqPlan {
  int first, n, len, blocks;       // first row, new tokens, tokens, query blocks
  int pos0;                        // slot of the first new token (below 0 where there are more than the sequence counts)
  int cost;                        // of a key
};

// Scratch of the plan in shared memory: only used before the first copy into the same memory.
struct PlanScratch {
  int64_t weight[kPlanMaxSeqs + 1];        // line at which each sequence starts
  int32_t units[kPlanMaxSeqs + 1];         // units before each sequence
  int32_t cut_unit[kPlanMaxBlocks + 1];    // where each block's range starts: the unit, and how far into it
  int64_t cut_off[kPlanMaxBlocks + 1];
  int64_t warp_w[kPlanThreads / 32];
  int64_t warp_u[kPlanThreads / 32];
};

struct Unit {
  SeqPlan s;
  int b, hk, block;
};

__device__ __forceinline__ SeqPlan seq_plan(const PlanParams& p, int b) {
  const int2 rows = new_rows(p.query_start, b, p.T);
  SeqPlan s;
  s.first = rows.x;
  s.n = rows.y - rows.x;
  s.len = table_len(p.kv_len, b, p.capacity);
  s.pos0 = first_slot(p.kv_len, b, s.n, p.capacity);
  s.blocks = (s.n + p.block_tokens - 1) / p.block_tokens;
  s.cost = s.n <= p.cheap_tokens ? kKeyCost : s.n <= p.tile_tokens ? p.cost_one : p.cost_two;
  return s;
}

// The same out of line, for the attention kernel: inlined in the dozen places of its plan, it costs the loops behind, which share the
// kernel's registers and instruction cache, 3% (2048 tokens x 40 heads over 61234 keys: 1970 us for 1915).
__device__ __attribute__((noinline)) inline SeqPlan seq_plan_apart(const PlanParams& p, int b) { return seq_plan(p, b); }

// Sum over j = 1 .. q of max(off + j * step, 0).
__device__ __forceinline__ int64_t ramp_sum(int64_t off, int64_t step, int64_t q) {
  const int64_t none = off >= 0 ? 0 : min(q, -off / step);
  return (q - none) * off + step * (q * (q + 1) - none * (none + 1)) / 2;
}

// What the first q query blocks of a sequence that is longer than its table have behind the table's end.
__device__ __attribute__((noinline)) inline int64_t past_length(const PlanParams& p, const SeqPlan& s, int q) {
  const int64_t over = static_cast<int64_t>(s.pos0) - s.len;
  const int64_t ends = ramp_sum(over, p.block_tokens, q);
  return p.window > 0 ? ends - ramp_sum(over - p.window + 1 - p.block_tokens, p.block_tokens, q) : ends;
}

// Weight of the first q query blocks of one head.
__device__ __forceinline__ int64_t head_weight(const PlanParams& p, const SeqPlan& s, int q) {
  int64_t w = static_cast<int64_t>(q) * kUnitCost;
  if (!p.causal) return (w + static_cast<int64_t>(q) * s.len) * s.cost;
  const int64_t before = s.pos0;
  w += ramp_sum(before, p.block_tokens, q);
  if (p.window > 0) w -= ramp_sum(before - p.window + 1 - p.block_tokens, p.block_tokens, q);
  if (before + s.n > s.len) w -= past_length(p, s, q);
  else if (q == s.blocks) w -= static_cast<int64_t>(q) * p.block_tokens - s.n;    // what the last block lacks
  return w * s.cost;
}

// Last i in [0, n) with a[i] <= x, where a[0] <= x.
template <class A>
__device__ __forceinline__ int last_at_most(const A* a, int n, int64_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (static_cast<int64_t>(a[mid]) <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ Unit unit_by_id(const PlanParams& p, const PlanScratch* sc, int id) {
  Unit u;
  u.b = last_at_most(sc->units, p.B, id);
  u.s = seq_plan_apart(p, u.b);
  const int rest = id - sc->units[u.b];
  u.hk = rest / u.s.blocks;
  u.block = rest - u.hk * u.s.blocks;
  return u;
}

// Place of a unit on the line, and its weight.
__device__ __forceinline__ int64_t unit_place(const PlanParams& p, const PlanScratch* sc, const Unit& u, int64_t& weight) {
  const int64_t before = head_weight(p, u.s, u.block);
  weight = head_weight(p, u.s, u.block + 1) - before;
  return sc->weight[u.b] + u.hk * head_weight(p, u.s, u.s.blocks) + before;
}

// The unit at place x of the line, 0 <= x < total; `off`: how far into it, `id`: its number.
__device__ __forceinline__ Unit unit_at(const PlanParams& p, const PlanScratch* sc, int64_t x, int64_t& off, int64_t& weight, int& id) {
  Unit u;
  u.b = last_at_most(sc->weight, p.B, x);
  u.s = seq_plan_apart(p, u.b);
  const int64_t head = head_weight(p, u.s, u.s.blocks);
  const int64_t rest = x - sc->weight[u.b];
  // a 64-bit division only where the numbers need it
  u.hk = ((rest | head) >> 32) == 0 ? static_cast<int>(static_cast<uint32_t>(rest) / static_cast<uint32_t>(head)) : static_cast<int>(rest / head);
  const int64_t in_head = rest - u.hk * head;
  u.block = 0;
  off = in_head;
  weight = head;
  if (u.s.blocks > 1) {
    int lo = 0, hi = u.s.blocks - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (head_weight(p, u.s, mid) <= in_head) lo = mid; else hi = mid - 1;
    }
    u.block = lo;
    const int64_t before = head_weight(p, u.s, lo);
    off = in_head - before;
    weight = head_weight(p, u.s, lo + 1) - before;
  }
  id = sc->units[u.b] + u.hk * u.s.blocks + u.block;
  return u;
}

// Unit that block i is dealt in round r: there and back, so that units that grow along the line even out.
__device__ __forceinline__ int dealt(int r, int i, int blocks) { return r * blocks + ((r & 1) ? blocks - 1 - i : i); }

// What a block sweeps of one unit.
struct Seg {
  int tok0, ntok;            // first row among the new tokens, and how many
  int hk;
  int b;
  int pos0;                  // slot of the first token, as a sequence's
  int len;
  int tile_begin, n_tiles;
  int slot;                  // >= 0: a piece, leaves its state in this slot
};

// Keys [x, y) that the token `i` behind a block's first one sees.
__device__ __forceinline__ int2 keys_of(const PlanParams& p, const Seg& s, int i) {
  if (!p.causal) return make_int2(0, s.len);
  const int hi = s.pos0 + i + 1;
  return make_int2(p.window > 0 ? max(hi - p.window, 0) : 0, min(max(hi, 0), s.len));
}

// Description of a whole unit.
__device__ __forceinline__ Seg whole_unit(const PlanParams& p, const SeqPlan& q, int b, int hk, int block) {
  Seg s;
  s.b = b;
  s.hk = hk;
  s.tok0 = q.first + block * p.block_tokens;
  s.ntok = min(p.block_tokens, q.n - block * p.block_tokens);
  s.pos0 = q.pos0 + block * p.block_tokens;
  s.len = q.len;
  s.slot = -1;
  const int lo = keys_of(p, s, 0).x, hi = keys_of(p, s, s.ntok - 1).y;
  s.tile_begin = lo / kPlanTile;
  s.n_tiles = hi > lo ? (hi + kPlanTile - 1) / kPlanTile - s.tile_begin : 0;
  return s;
}

// The part of unit u from `a` on, as far as `e` unless `to_end`, in the line's measure.
__device__ __forceinline__ Seg part_of_unit(const PlanParams& p, const Unit& u, int64_t a, int64_t e, bool to_end, int me) {
  Seg s = whole_unit(p, u.s, u.b, u.hk, u.block);
  const bool begins = a == 0;
  if (begins && to_end) return s;
  const int64_t n = s.n_tiles;
  a /= u.s.cost;
  e /= u.s.cost;
  const int64_t from = a <= kUnitCost ? 0 : min((a - kUnitCost) / kPlanTile, n);
  const int64_t to = to_end ? n : e <= kUnitCost ? 0 : min((e - kUnitCost) / kPlanTile, n);
  s.slot = 2 * me + (begins ? 1 : 0);
  s.tile_begin += static_cast<int>(from);
  s.n_tiles = static_cast<int>(to - from);
  return s;
}

// The unit behind u = (sequence, key head, query block) on the line; q is its sequence's.
__device__ __forceinline__ void next_unit(const PlanParams& p, SeqPlan& q, int3& u) {
  if (++u.z < q.blocks) return;
  u.z = 0;
  if (++u.y < p.Hkv) return;
  u.y = 0;
  while (u.x + 1 < p.B) {
    q = seq_plan_apart(p, ++u.x);
    if (q.blocks > 0) return;
  }
}

struct BlockPlan {
  int rounds;              // whole units dealt to every block
  int first_unit, n_units; // units of this block's range
  int64_t begin, end;      // how far into its first unit it begins, and into its last one it ends; end 0: at its end
  // Part of the i-th unit of the range.
  __device__ __forceinline__ Seg part(const PlanParams& p, const Unit& u, int i, int me) const {
    return part_of_unit(p, u, i == 0 ? begin : 0, end, i < n_units - 1 || end == 0, me);
  }
  // The last unit begins here and goes on in the next blocks' ranges.
  __device__ __forceinline__ bool opens() const { return n_units > 0 && end > 0 && (n_units > 1 || begin == 0); }
};

// Pieces of the unit that block `me`'s range opens: of the cuts behind, those that lie in it, and one.
__device__ __forceinline__ int pieces_of(const PlanScratch* sc, const BlockPlan& bp, int blocks, int me) {
  return 1 + last_at_most(sc->cut_unit + me, blocks - me, bp.first_unit + bp.n_units - 1);
}

// Fills the scratch; called by all kPlanThreads threads.  Returns the rounds of whole units, -1 where there is no unit at
// all, or more than an int can number.  Sequences without new tokens take no room on the line, and the searches land on the last of several that start at the
// same place: the one that has some.
__device__ __forceinline__ int make_cuts(const PlanParams& p, PlanScratch* sc, int blocks) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // in the high bits of the unit count: sequences that have any (8192 times the rows of any tensor stay below)
  constexpr int kSeqBit = 45;
  int64_t base_w = 0, base_u = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int64_t w = 0, u = 0;
    if (b < p.B) {
      const SeqPlan s = seq_plan_apart(p, b);
      if (s.blocks > 0) {
        w = p.Hkv * head_weight(p, s, s.blocks);
        u = static_cast<int64_t>(s.blocks) * p.Hkv + (1ll << kSeqBit);
      }
    }
    int64_t iw = w, iu = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t yw = __shfl_up_sync(0xffffffffu, iw, o), yu = __shfl_up_sync(0xffffffffu, iu, o);
      if (lane >= o) { iw += yw; iu += yu; }
    }
    if (lane == 31) { sc->warp_w[warp] = iw; sc->warp_u[warp] = iu; }
    __syncthreads();
    int64_t pw = base_w, pu = base_u;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 32; ++i) {
      if (i < warp) { pw += sc->warp_w[i]; pu += sc->warp_u[i]; }
      base_w += sc->warp_w[i];
      base_u += sc->warp_u[i];
    }
    if (b < p.B) {
      sc->weight[b] = pw + iw - w;
      sc->units[b] = static_cast<int32_t>((pu + iu - u) & 0xffffffff);
    }
    __syncthreads();
  }
  const int64_t total = base_w;
  const int64_t all_units = base_u & ((1ll << kSeqBit) - 1);
  if (all_units == 0 || all_units > 0x7fffffff) return -1;   // too many only where query_start gives rows to several sequences
  const int units = static_cast<int>(all_units);
  const int seqs = static_cast<int>(base_u >> kSeqBit);
  int rounds = 0;
  if (units >= blocks && units >= 2 * seqs * p.Hkv && total / units >= static_cast<int64_t>(kLongUnit) * kKeyCost) rounds = min(units / blocks, kPlanMaxRounds);
  int64_t start = 0, share = 0;
  if (rounds > 0) {
    const int64_t mean = (total + blocks - 1) / blocks;
    for (;;) {
      int64_t load = 0;
      if (tid < blocks)
        for (int r = 0; r < rounds; ++r) {
          int64_t w;
          unit_place(p, sc, unit_by_id(p, sc, dealt(r, tid, blocks)), w);
          load += w;
        }
      // a deal that gives a block 2% more than its part of everything leaves too little to even out
      const int over = __syncthreads_or(load > mean + mean / 50);
      if (!over || rounds == 1) {
        int64_t w;
        start = rounds * blocks < units ? unit_place(p, sc, unit_by_id(p, sc, rounds * blocks), w) : total;
        share = max(mean - load, static_cast<int64_t>(start < total ? kUnitCost * kKeyCost : 0));
        break;
      }
      --rounds;
    }
  } else {
    share = max((total + blocks - 1) / blocks, static_cast<int64_t>(kUnitCost * kKeyCost));
  }
  // where each range starts: the shares before it
  {
    int64_t x = tid < blocks ? share : 0, inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sc->warp_w[warp] = inc;
    __syncthreads();
    int64_t before = start;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 32; ++i)
      if (i < warp) before += sc->warp_w[i];
    if (tid < blocks) {
      const int64_t cut = before + inc - x;
      int id = cut <= start ? rounds * blocks : units;
      int64_t off = 0;
      if (cut > start && cut < total) {
        int64_t weight;
        const int cost = unit_at(p, sc, cut, off, weight, id).s.cost;
        if (off < (kUnitCost + kLeastKeys) * cost) {
          off = 0;
        } else if (weight - off < kLeastKeys * cost) {
          off = 0;
          ++id;
        }
      }
      sc->cut_unit[tid] = id;
      sc->cut_off[tid] = off;
    }
    if (tid == 0) {
      sc->cut_unit[blocks] = units;
      sc->cut_off[blocks] = 0;
    }
    __syncthreads();
  }
  return rounds;
}

// Block `me`'s part of the plan.
__device__ __forceinline__ BlockPlan make_plan(const PlanParams& p, PlanScratch* sc, int blocks, int me) {
  BlockPlan bp = {0, 0, 0, 0, 0};
  const int rounds = make_cuts(p, sc, blocks);
  if (rounds < 0) return bp;
  bp.rounds = rounds;
  bp.first_unit = sc->cut_unit[me];
  bp.begin = sc->cut_off[me];
  bp.end = sc->cut_off[me + 1];
  bp.n_units = sc->cut_unit[me + 1] - bp.first_unit + (bp.end > 0 ? 1 : 0);
  return bp;
}

// What a block keeps of its plan once the scratch is gone: all that the units behind the first few are described from.
struct BlockUnits {
  int3 dealt[kPlanMaxRounds];      // sequence, key head, query block
  int3 start;                      // of the range's first unit
  Seg first, last;                 // of the range: the two units of it that may be swept in part
};

// Descriptions of the first n < kPlanThreads units of block `me` go to `segs`, and what the others' are made from to `units`.  Where
// the block opens its last unit, the thread that described that gets the number of its pieces back; all others get 0.
__device__ __forceinline__ int first_units(const PlanParams& p, const PlanScratch* sc, const BlockPlan& bp, int blocks, int me, BlockUnits& units,
                                           Seg* segs, int n) {
  const int i = threadIdx.x;
  for (int r = i; r < bp.rounds; r += kPlanThreads) {
    const Unit u = unit_by_id(p, sc, dealt(r, me, blocks));
    units.dealt[r] = make_int3(u.b, u.hk, u.block);
    if (r < n) segs[r] = whole_unit(p, u.s, u.b, u.hk, u.block);
  }
  // the first units of the range, and, a thread behind those, its last
  const int of_range = min(bp.n_units, n);
  if (bp.n_units == 0 || (i >= of_range && i != n)) return 0;
  const int k = i < of_range ? i : bp.n_units - 1;
  const Unit u = unit_by_id(p, sc, bp.first_unit + k);
  const Seg s = bp.part(p, u, k, me);
  if (i < of_range && bp.rounds + i < n) segs[bp.rounds + i] = s;
  if (i == 0) {
    units.start = make_int3(u.b, u.hk, u.block);
    units.first = s;
  }
  if (i != n) return 0;
  units.last = s;
  return bp.opens() ? pieces_of(sc, bp, blocks, me) : 0;
}

// The units of a block from number `from` on, one at a time.
struct UnitWalk {
  int i, rounds, total;
  int3 u;                          // of the range: its first unit's until i is behind it
  SeqPlan q;
  __device__ __forceinline__ UnitWalk(const PlanParams& p, const BlockUnits& units, int rounds, int total, int from)
      : i(from), rounds(rounds), total(total), u(units.start) {
    if (total == rounds) return;                         // no range
    q = seq_plan_apart(p, u.x);
    for (int k = rounds; k < from && k + 1 < total; ++k) next_unit(p, q, u);
  }
  __device__ __forceinline__ bool more() const { return i < total; }
  __device__ __forceinline__ Seg seg(const PlanParams& p, const BlockUnits& units) const {
    if (i < rounds) {
      const int3 d = units.dealt[i];
      return whole_unit(p, seq_plan_apart(p, d.x), d.x, d.y, d.z);
    }
    return i == total - 1 ? units.last : i == rounds ? units.first : whole_unit(p, q, u.x, u.y, u.z);
  }
  __device__ __forceinline__ void next(const PlanParams& p) {
    if (i >= rounds && i + 1 < total) next_unit(p, q, u);
    ++i;
  }
};

}  // namespace dtb
