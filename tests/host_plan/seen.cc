// Reads calls (as plan.cc) and prints, a line each, the keys [x, y) that each new token sees, of all sequences in order; checks that a
// query block weighs the keys that its tokens see together.
#include <cstdio>
#include <cstdlib>
#include <iostream>

#include "paged_plan.cuh"

using namespace dtb;

int main() {
  PlanParams p;
  int blocks;
  for (; std::cin >> p.causal >> p.window >> p.block_tokens >> p.Hkv >> blocks >> p.capacity >> p.T >> p.B;) {
    std::vector<int32_t> starts(p.B + 1), lens(p.B);
    for (auto& x : starts) std::cin >> x;
    for (auto& x : lens) std::cin >> x;
    p.query_start = starts.data();
    p.kv_len = lens.data();
    for (int b = 0; b < p.B; ++b) {
      const SeqPlan q = seq_plan(p, b);
      for (int block = 0; block < q.blocks; ++block) {
        const Seg s = whole_unit(p, q, b, 0, block);
        for (int i = 0; i < s.ntok; ++i) {
          const int2 k = keys_of(p, s, i);
          std::printf("%d %d ", k.x, k.y);
        }
        const int64_t keys = std::max(keys_of(p, s, s.ntok - 1).y - keys_of(p, s, 0).x, 0), weight = head_weight(p, q, block + 1) - head_weight(p, q, block);
        if (weight != (kUnitCost + keys) * q.cost) {
          std::printf("\nblock %d of sequence %d weighs %lld for %lld keys\n", block, b, (long long)weight, (long long)keys);
          return 1;
        }
      }
    }
    std::printf("\n");
  }
  return 0;
}
