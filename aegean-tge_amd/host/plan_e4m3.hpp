// Planning of a step on an e4m3 pool: append tiles and attention items.
#pragma once

#include <vector>

#include "../csrc/e4m3_common.h"
#include "plan.hpp"

namespace tge::plan {

struct E4m3Lists {
  std::vector<E4m3Tile> tiles;
  bool page_twice = false;  // two sessions append into one page
  std::vector<E4m3Item> items;  // workgroup i starts with item i
  std::vector<E4m3Merge> merges;
  int groups = 0;
  int parts = 0;      // partial states
  int part_rows = 32; // rows of each
};

// `cus` compute units, each holding `per_cu` workgroups at once.
void build_e4m3(const Step& s, int cus, int per_cu, E4m3Lists& out);

}  // namespace tge::plan
