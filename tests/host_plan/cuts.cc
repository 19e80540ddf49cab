// Reads calls (as plan.cc) and prints of each what make_cuts returns, and the number of units that it counts.
#include <cstdio>
#include <iostream>

#include "paged_plan.cuh"

using namespace dtb;

int main() {
  PlanParams p;
  int blocks;
  std::barrier<> all(kPlanThreads);
  block_barrier = &all;
  for (int i = 0; i < kPlanThreads / 32; ++i) warp_barriers.push_back(new std::barrier<>(32));
  auto* sc = new PlanScratch;
  for (; std::cin >> p.causal >> p.window >> p.block_tokens >> p.Hkv >> blocks >> p.capacity >> p.T >> p.B;) {
    std::vector<int32_t> starts(p.B + 1), lens(p.B);
    for (auto& x : starts) std::cin >> x;
    for (auto& x : lens) std::cin >> x;
    p.query_start = starts.data();
    p.kv_len = lens.data();
    int rounds = 0;
    std::vector<std::thread> threads;
    for (int t = 0; t < kPlanThreads; ++t)
      threads.emplace_back([&, t] {
        threadIdx.x = t;
        const int r = make_cuts(p, sc, blocks);
        if (t == 0) rounds = r;
      });
    for (auto& t : threads) t.join();
    std::printf("%d %d\n", rounds, rounds < 0 ? 0 : sc->cut_unit[blocks]);
  }
}
