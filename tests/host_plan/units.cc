// Reads calls (as plan.cc) and walks the units of every block as the attention kernel does: the first kSegs described by the
// block's threads, the others by one warp from what the block has kept.  Together they have to sweep every key tile of every unit
// once, a unit that is swept in pieces has to leave each of them in the slot where the merge looks for it, and the block that opens
// it has to have counted them.
#include <cstdio>
#include <cstdlib>
#include <iostream>
#include <map>
#include <tuple>

#include "paged_plan.cuh"

using namespace dtb;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (call %d)\n", __LINE__, #x, call); std::exit(1); } } while (0)

int main() {
  int call = 0;
  PlanParams p;
  int blocks;
  std::barrier<> all(kPlanThreads);
  block_barrier = &all;
  for (int i = 0; i < kPlanThreads / 32; ++i) warp_barriers.push_back(new std::barrier<>(32));
  auto* sc = new PlanScratch;
  for (; std::cin >> p.causal >> p.window >> p.block_tokens >> p.Hkv >> blocks >> p.capacity >> p.T >> p.B; ++call) {
    std::vector<int32_t> starts(p.B + 1), lens(p.B);
    for (auto& x : starts) std::cin >> x;
    for (auto& x : lens) std::cin >> x;
    p.cheap_tokens = p.tile_tokens = p.block_tokens / 2;
    p.cost_two = 11;
    p.query_start = starts.data();
    p.kv_len = lens.data();
    int rounds = 0;
    {
      std::vector<std::thread> threads;
      for (int t = 0; t < kPlanThreads; ++t)
        threads.emplace_back([&, t] {
          threadIdx.x = t;
          const int r = make_cuts(p, sc, blocks);
          if (t == 0) rounds = r;
        });
      for (auto& t : threads) t.join();
    }
    if (rounds < 0) continue;
    int behind = 0;                        // blocks whose range begins in a unit that the warp describes, and in the middle of it
    for (const int held : {16, 3}) {
      std::map<std::tuple<int, int, int>, std::vector<Seg>> swept;
      std::map<std::tuple<int, int, int>, int> counted;          // unit -> its pieces, as the block says that opens it
      for (int me = 0; me < blocks; ++me) {
        BlockPlan bp = {rounds, sc->cut_unit[me], 0, sc->cut_off[me], sc->cut_off[me + 1]};      // as make_plan ends
        bp.n_units = sc->cut_unit[me + 1] - bp.first_unit + (bp.end > 0 ? 1 : 0);
        const int total = bp.rounds + bp.n_units;
        BlockUnits units;
        std::vector<Seg> segs(held, Seg{-1, -1, -1, -1, -1, -1, -1, -1, -1});
        int pieces = 0;
        for (int t = 0; t < kPlanThreads; ++t) {
          threadIdx.x = t;
          if (const int n = first_units(p, sc, bp, blocks, me, units, segs.data(), held)) {
            CHECK(pieces == 0);
            pieces = n;
          }
        }
        CHECK((pieces > 0) == bp.opens());
        segs.resize(std::min(total, held));
        for (UnitWalk w(p, units, bp.rounds, total, held); w.more(); w.next(p)) {
          CHECK(w.i == static_cast<int>(segs.size()));
          segs.push_back(w.seg(p, units));
        }
        CHECK(static_cast<int>(segs.size()) == total);
        behind += held == 16 && bp.rounds >= held && bp.begin > 0 && bp.n_units > 1;
        for (int i = 0; i < total; ++i) {
          const Seg& s = segs[i];
          CHECK(s.b >= 0 && s.b < p.B && s.hk >= 0 && s.hk < p.Hkv && s.ntok > 0);
          const int first = seq_plan(p, s.b).first;
          CHECK((s.tok0 - first) % p.block_tokens == 0);
          const std::tuple<int, int, int> unit = {s.b, s.hk, (s.tok0 - first) / p.block_tokens};
          if (s.slot >= 0) CHECK(s.slot / 2 == me);
          swept[unit].push_back(s);
          if (i == total - 1 && pieces > 0) counted[unit] = pieces;
        }
      }
      int64_t n_units = 0;
      for (int b = 0; b < p.B; ++b) n_units += static_cast<int64_t>(seq_plan(p, b).blocks) * p.Hkv;
      CHECK(static_cast<int64_t>(swept.size()) == n_units);
      for (auto& [unit, parts] : swept) {
        auto [b, hk, block] = unit;
        const Seg w = whole_unit(p, seq_plan(p, b), b, hk, block);
        int tile = w.tile_begin;
        for (const Seg& s : parts) {
          CHECK(s.tile_begin == tile || s.n_tiles == 0);
          CHECK(s.tok0 == w.tok0 && s.ntok == w.ntok && s.pos0 == w.pos0 && s.len == w.len);
          tile += s.n_tiles;
        }
        CHECK(tile == w.tile_begin + w.n_tiles);
        if (parts.size() == 1) {
          CHECK(parts[0].slot == -1 && counted.count(unit) == 0);
          continue;
        }
        CHECK(counted.count(unit) && counted[unit] == static_cast<int>(parts.size()));
        const int k = parts[0].slot / 2;
        for (size_t i = 0; i < parts.size(); ++i) CHECK(parts[i].slot == static_cast<int>(i == 0 ? 2 * k + 1 : 2 * (k + i)));
      }
    }
    std::printf("%d rounds, %d ranges begin inside a unit behind the first 16\n", rounds, behind);
  }
  return 0;
}
