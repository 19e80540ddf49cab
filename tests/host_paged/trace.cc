// Prints what representative threads of one block of the paged attention kernel do over a batch that it has to itself:
// trace DIM KERNEL MODE G WARPS new:kv ...
//   KERNEL  thin (units of few rows with keys as rows) or thick
//   MODE    steady, or growing (the offset moves at every tile)
#include <string>

#include "paged_plan.cuh"

namespace dtb {
BlockPlan host_plan(PlanScratch* scratch);
}
#include "paged_attn.cuh"

Index3 threadIdx, blockIdx, gridDim = {1, 1, 1};

using namespace dtb;

static PagedKernelParams p;
static BlockPlan plan;
static PlanScratch filled;
static std::function<void()> describe_first;

// The plan of a single block, which takes all units, and the descriptions that the block's threads make of the first ones.
BlockPlan dtb::host_plan(PlanScratch* scratch) {
  *scratch = filled;
  describe_first();
  return plan;
}

template <int kD, bool kThin>
void trace(bool grow, int warps) {
  using Bars = PagedBarriers<kD>;
  auto* bars = reinterpret_cast<Bars*>(smem_raw + 2 * 128 * kD * 2 + kRingBytes);
  const int total = plan.rounds + plan.n_units;
  std::vector<Seg> all;
  std::vector<int> waited(kSegs);
  describe_first = [&] {
    const Index3 me = threadIdx;
    for (unsigned t = 0; t < kPlanThreads; ++t) {
      threadIdx.x = t;
      first_units(p.plan, &filled, plan, 1, 0, bars->units, bars->segs, kSegs);
    }
    threadIdx = me;
    all.assign(bars->segs, bars->segs + std::min(total, kSegs));
    for (UnitWalk w(p.plan, bars->units, plan.rounds, total, kSegs); w.more(); w.next(p.plan)) all.push_back(w.seg(p.plan, bars->units));
  };
  describe = [&](uint32_t bar) {
    for (int i = 0; i < kSegs; ++i)
      if (bar == smem_u32(&bars->seg_full[i])) bars->segs[i] = all.at(kSegs * ++waited[i] + i);
  };
  auto run = [&](const std::string& role, int thread) {
    std::memset(smem_raw, 0, sizeof(smem_raw));
    waited.assign(kSegs, 0);
    threadIdx = {static_cast<unsigned>(thread), 0, 0};
    growing = grow;
    tiles_read = 0;
    std::printf("thread %s\n", role.c_str());
    paged_attn_kernel<__nv_bfloat16, kD, kThin>(p);
  };
  run("load", kLoadWarp * 32);
  run("scores", kMmaWarp * 32);
  run("values", kPvWarp * 32);
  run("units", (kPvWarp + 1) * 32);
  for (int group = 0; group < 2; ++group)
    for (int w = 0; w < warps; ++w) run("group" + std::to_string(group) + "." + std::to_string(w), group * kBlockM + 32 * w);

  auto name = [&](const char* what, const uint64_t& bar) { std::printf("name %u %s\n", smem_u32(&bar), what); };
  for (int i = 0; i < Bars::kSlots; ++i) { name("kv_full", bars->kv_full[i]); name("kv_empty", bars->kv_empty[i]); }
  for (int i = 0; i < kSegs; ++i) { name("seg_full", bars->seg_full[i]); name("seg_empty", bars->seg_empty[i]); }
  for (int t = 0; t < 2; ++t) { name("s_full", bars->s_full[t]); name("p_lo", bars->p_lo[t]); name("p_hi", bars->p_hi[t]); name("pv_done", bars->pv_done[t]); }
  for (auto* bar = reinterpret_cast<const uint64_t*>(&bars->o_free); bar != reinterpret_cast<const uint64_t*>(&bars->o_free + 1); ++bar) name("o_free", *bar);
  name("q_full", bars->q_full); name("q_empty", bars->q_empty); name("s_free", bars->s_free); name("vote", bars->vote);
}

int main(int argc, char** argv) {
  if (argc < 7) return 2;
  const int D = std::atoi(argv[1]), G = std::atoi(argv[4]), warps = std::atoi(argv[5]), B = argc - 6;
  const bool thin = argv[2] == std::string("thin"), grow = argv[3] == std::string("growing");
  std::vector<int32_t> starts(1), lens;
  for (int b = 0; b < B; ++b) {
    const std::string s = argv[6 + b];
    const size_t colon = s.find(':');
    starts.push_back(starts.back() + std::stoi(s.substr(0, colon)));
    lens.push_back(std::stoi(s.substr(colon + 1)));
  }
  const int T = starts.back(), capacity = 4096;
  std::vector<int32_t> table(B * capacity / 64);
  std::vector<__nv_bfloat16> o(static_cast<size_t>(T) * G * D);
  MergeDesc merge;
  p.tmap_q.name = 'Q'; p.tmap_k.name = 'K'; p.tmap_v.name = 'V';
  p.G = p.Hq = G;
  p.tile_tokens = kBlockM / G;
  p.plan = {starts.data(), lens.data(), capacity, B, T, 1, 2 * p.tile_tokens, 1, 0};
  p.page_table = table.data();
  p.table_stride = p.table_width = capacity / 64;
  p.pages = 1;
  p.page_size = 64;
  p.o = o.data();
  p.o_stride_t = G * D;
  p.o_stride_h = D;
  p.merge = &merge;
  p.scale_log2 = 1.f;
  int64_t weight = 0;
  for (int b = 0; b < B; ++b) {
    const SeqPlan s = seq_plan(p.plan, b);
    filled.weight[b] = weight;
    filled.units[b] = plan.n_units;
    weight += s.blocks > 0 ? head_weight(p.plan, s, s.blocks) : 0;
    plan.n_units += s.blocks;
  }
  filled.cut_unit[1] = plan.n_units;
  if (D == 128) thin ? trace<128, true>(grow, warps) : trace<128, false>(grow, warps);
  else thin ? trace<64, true>(grow, warps) : trace<64, false>(grow, warps);
}
