// Reads calls (one a line: causal window block_tokens Hkv blocks page_capacity T B, then B + 1 starts and B lengths) and checks the plan
// of each: every block's pieces, in bounds and in the order in which the kernel walks them, cover every key tile of every
// unit exactly once, pieces of a unit lie in the slots where the merge looks for them, and no other slot is used.
#include <cstdio>
#include <cstdlib>
#include <iostream>
#include <map>
#include <set>
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
    // every other call with units whose keys cost differently
    p.cheap_tokens = call & 1 ? 3 : 0;
    p.tile_tokens = call & 1 ? p.block_tokens / 2 : 0;
    p.cost_one = call & 1 ? 12 : kKeyCost;
    p.cost_two = call & 1 ? 16 : kKeyCost;
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
    std::map<std::tuple<int, int, int>, std::vector<Seg>> swept;   // unit -> its parts, in the order of the blocks
    int64_t units = 0, heaviest = 0, whole = 0;
    for (int b = 0; b < p.B; ++b) units += static_cast<int64_t>(seq_plan(p, b).blocks) * p.Hkv;
    CHECK((rounds < 0) == (units == 0));
    std::map<int, std::pair<int, std::tuple<int, int, int>>> merges;   // first block -> pieces and unit
    int widest = 0;
    for (int me = 0; rounds >= 0 && me < blocks; ++me) {
      CHECK(sc->cut_unit[me] <= sc->cut_unit[me + 1] && rounds <= kPlanMaxRounds);
      CHECK(sc->cut_unit[me] < sc->cut_unit[me + 1] || sc->cut_off[me] <= sc->cut_off[me + 1]);
      int64_t load = 0;
      int parts = 0;
      auto note = [&](int b, int hk, int block, const Seg& s) {
        CHECK(b >= 0 && b < p.B && hk >= 0 && hk < p.Hkv && block >= 0 && block < seq_plan(p, b).blocks);
        CHECK(s.b == b && s.hk == hk && s.ntok > 0 && s.tok0 >= 0 && s.tok0 + s.ntok <= p.T && s.n_tiles >= 0 && s.tile_begin >= 0);
        swept[{b, hk, block}].push_back(s);
        load += s.n_tiles;
        ++parts;
      };
      for (int r = 0; r < rounds; ++r) {
        const Unit u = unit_by_id(p, sc, dealt(r, me, blocks));
        note(u.b, u.hk, u.block, whole_unit(p, u.s, u.b, u.hk, u.block));
      }
      BlockPlan bp = {rounds, sc->cut_unit[me], 0, sc->cut_off[me], sc->cut_off[me + 1]};      // as make_plan ends
      bp.n_units = sc->cut_unit[me + 1] - bp.first_unit + (bp.end > 0 ? 1 : 0);
      if (bp.n_units > 0) {
        const Unit f = unit_by_id(p, sc, bp.first_unit);
        int3 at = {f.b, f.hk, f.block};
        SeqPlan q = seq_plan(p, at.x);
        for (int i = 0; i < bp.n_units; ++i) {
          const Unit u = unit_by_id(p, sc, bp.first_unit + i);
          CHECK(u.b == at.x && u.hk == at.y && u.block == at.z);
          int64_t weight, off, w2;
          int id;
          const int64_t place = unit_place(p, sc, u, weight);
          for (int64_t x : {int64_t{0}, weight - 1}) {
            const Unit v = unit_at(p, sc, place + x, off, w2, id);
            CHECK(v.b == u.b && v.hk == u.hk && v.block == u.block && off == x && w2 == weight && id == bp.first_unit + i);
          }
          const Seg s = bp.part(p, u, i, me);
          if (i != 0 && i != bp.n_units - 1) {          // the kernel takes those between for whole
            const Seg w = whole_unit(p, u.s, u.b, u.hk, u.block);
            CHECK(s.slot == -1 && s.tile_begin == w.tile_begin && s.n_tiles == w.n_tiles);
          }
          note(u.b, u.hk, u.block, s);
          if (i < bp.n_units - 1) next_unit(p, q, at);
        }
        if (bp.opens()) {
          const Unit l = unit_by_id(p, sc, bp.first_unit + bp.n_units - 1);
          merges[me] = {pieces_of(sc, bp, blocks, me), {l.b, l.hk, l.block}};
        }
      }
      heaviest = std::max(heaviest, load);
      whole += load;
      widest = std::max(widest, parts);
    }
    CHECK(static_cast<int64_t>(swept.size()) == units);
    std::set<int> slots;
    size_t pieces = 0;
    for (auto& [unit, parts] : swept) {
      auto [b, hk, block] = unit;
      const SeqPlan q = seq_plan(p, b);
      const Seg w = whole_unit(p, q, b, hk, block);
      int tile = w.tile_begin;
      for (const Seg& s : parts) {
        CHECK(s.tile_begin == tile || s.n_tiles == 0);
        tile += s.n_tiles;
        CHECK(s.tok0 == w.tok0 && s.ntok == w.ntok && s.pos0 == w.pos0 && s.len == w.len);
      }
      CHECK(tile == w.tile_begin + w.n_tiles);
      if (parts.size() == 1) {
        CHECK(parts[0].slot == -1);
        continue;
      }
      const int k = parts[0].slot / 2;
      CHECK(parts[0].slot == 2 * k + 1 && merges.count(k) && merges[k].second == unit && merges[k].first == static_cast<int>(parts.size()));
      for (size_t i = 1; i < parts.size(); ++i) CHECK(parts[i].slot == static_cast<int>(2 * (k + i)) && k + static_cast<int>(i) < blocks);
      for (const Seg& s : parts) CHECK(slots.insert(s.slot).second);
      ++pieces;
    }
    CHECK(merges.size() == pieces);
    std::printf("%d rounds, %lld units, %zu of them cut, heaviest block %lld of %lld tiles, %d parts at most\n", rounds, (long long)units, pieces,
                (long long)heaviest, (long long)whole, widest);
  }
  return 0;
}
