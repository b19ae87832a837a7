// Prints what the plan of a step on an e4m3 pool holds (aegean-tge_amd/host/
// plan_e4m3.cpp): arguments query heads, KV heads, head_dim, then ctx and new
// tokens of each session. Built with the sanitizers and run by
// tests/test_e4m3_plans.py, which pins the plans of the GPU tests' steps.
//   items, groups   work items and workgroups
//   chained         items that are not their workgroup's first
//   unlike          workgroups whose items differ in rows of a tile or session
//   rw1, rw2, rw4   items by waves of rows
//   cut             items that are a piece of a cut tile; most: pieces of a tile
//   longest         pages of the longest item
//   outgrown        merges whose states' bases and sums the LDS ring cannot hold
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../aegean-tge_amd/host/plan_e4m3.hpp"
#include "tge_kv.h"

int main(int argc, char** argv) {
  if (argc < 6 || argc % 2 != 0) return 1;
  std::vector<int> a;
  for (int i = 1; i < argc; ++i) a.push_back(std::atoi(argv[i]));
  std::vector<int> ctx, n_new, offsets{0};
  for (std::size_t i = 3; i < a.size(); i += 2) {
    ctx.push_back(a[i]);
    n_new.push_back(a[i + 1]);
    offsets.push_back(offsets.back() + (a[i] + a[i + 1] + 15) / 16);
  }
  const std::vector<int> ids((std::size_t)offsets.back(), 0);
  tge::plan::Step st;
  const char* msg = "";
  if (tge::plan::build_step(st, (int)ctx.size(), ctx.data(), n_new.data(), offsets.data(), ids.data(), a[0], a[1], a[2],
                            1, &msg) != TGE_OK) {
    std::printf("%s\n", msg);
    return 1;
  }
  tge::plan::E4m3Lists l;
  tge::plan::build_e4m3(st, 256, a[2] > 128 ? 1 : a[2] > 64 ? 2 : 3, l);
  int rw[5] = {}, cut = 0, most = 0, longest = 0, outgrown = 0, unlike = 0;
  for (const auto& it : l.items) {
    ++rw[it.rw];
    cut += it.part >= 0;
    longest = std::max(longest, it.page_end - it.page_begin);
  }
  for (const auto& m : l.merges) {
    most = std::max(most, m.n_parts);
    outgrown += m.n_parts * m.rows * 8 > 16 * tge::e4m3_block_bytes(st.block_dims);
  }
  for (int g = 0; g < l.groups; ++g) {
    bool differ = false;
    const auto& first = l.items[(std::size_t)g];
    for (int i = first.next; i >= 0; i = l.items[(std::size_t)i].next)
      differ = differ || l.items[(std::size_t)i].rows != first.rows || l.items[(std::size_t)i].table_off != first.table_off;
    unlike += differ;
  }
  std::printf("items %zu groups %d chained %d unlike %d rw1 %d rw2 %d rw4 %d cut %d most %d longest %d outgrown %d\n",
              l.items.size(), l.groups, (int)l.items.size() - l.groups, unlike, rw[1], rw[2], rw[4], cut, most, longest,
              outgrown);
  return 0;
}
