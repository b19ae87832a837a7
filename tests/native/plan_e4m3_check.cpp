// Host check of the e4m3 plans (aegean-tge_amd/host/plan_e4m3.cpp), built with
// the address and undefined-behaviour sanitizers by tests/test_e4m3.py.
//   - every new row of every session is in one append tile, with its page and
//     slot; a page that two sessions append into is reported;
//   - the items of every (session, KV head) cover each of its rows once, and
//     every row's visible pages exactly once;
//   - every item is reached from one workgroup, once; the pieces of a cut tile
//     own the partial slots of its merge record, in the order of their pages;
//   - partial states stay below the 2 GiB that the kernel addresses.
// With arguments (query heads, KV heads, head_dim, ctx, new tokens, sessions)
// it prints what that plan holds instead.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "../../aegean-tge_amd/host/plan_e4m3.hpp"
#include "tge_kv.h"

using namespace tge;
using namespace tge::plan;

#define REQUIRE(c, ...)                                        \
  do {                                                         \
    if (!(c)) {                                                \
      std::printf("FAIL %s:%d: %s: ", __FILE__, __LINE__, #c); \
      std::printf(__VA_ARGS__);                                \
      std::printf("\n");                                       \
      std::exit(1);                                            \
    }                                                          \
  } while (0)

namespace {

struct Desc {
  std::vector<int> ctx, n_new, offsets{0}, ids;
  void add(int c, int n, int pool_pages, std::mt19937& rng) {
    ctx.push_back(c);
    n_new.push_back(n);
    for (int i = 0; i < (c + n + 15) / 16; ++i) ids.push_back((int)(rng() % pool_pages));
    offsets.push_back((int)ids.size());
  }
};

Step step_of(const Desc& d, int q_heads, int kv_heads, int head_dim, int pool_pages) {
  Step st;
  const char* msg = "";
  const int s = build_step(st, (int)d.ctx.size(), d.ctx.data(), d.n_new.data(), d.offsets.data(), d.ids.data(), q_heads,
                           kv_heads, head_dim, pool_pages, &msg);
  REQUIRE(s == TGE_OK, "%s", msg);
  return st;
}

void check_append(const Step& st, const E4m3Lists& l) {
  std::map<int, int> uses;
  std::size_t at = 0;
  int row = 0;
  for (const SessionRec& r : st.sessions)
    for (int pos = r.ctx; pos < r.ctx + r.n_new;) {
      REQUIRE(at < l.tiles.size(), "%zu tiles", at);
      const E4m3Tile& t = l.tiles[at++];
      REQUIRE(t.pos == pos && t.row == row && t.slot == pos % 16, "tile %zu", at - 1);
      REQUIRE(t.page == st.tables[(std::size_t)(r.table_off + pos / 16)], "page of tile %zu", at - 1);
      REQUIRE(t.count >= 1 && t.slot + t.count <= 16 && pos + t.count <= r.ctx + r.n_new, "count %d", t.count);
      REQUIRE(t.slot + t.count == 16 || pos + t.count == r.ctx + r.n_new, "a page is one tile");
      ++uses[t.page];
      pos += t.count;
      row += t.count;
    }
  REQUIRE(at == l.tiles.size(), "tiles left");
  bool twice = false;
  for (const auto& u : uses) twice = twice || u.second > 1;
  REQUIRE(twice == l.page_twice, "page_twice %d", l.page_twice);
}

void check_attention(const Step& st, const E4m3Lists& l) {
  // every item once
  std::vector<int> reached(l.items.size(), 0);
  REQUIRE(l.groups >= 1 && l.groups <= (int)l.items.size(), "groups %d", l.groups);
  for (int g = 0; g < l.groups; ++g)
    for (int i = g; i >= 0; i = l.items[(std::size_t)i].next) {
      REQUIRE(i < (int)l.items.size(), "item %d", i);
      REQUIRE(reached[(std::size_t)i]++ == 0, "item %d twice", i);
    }
  REQUIRE(std::count(reached.begin(), reached.end(), 1) == (long)reached.size(), "items left");
  REQUIRE((long long)l.parts * l.part_rows * st.block_dims * 4 < (1LL << 31), "%d parts", l.parts);
  // (table, KV head, first row) -> items
  std::map<std::tuple<int, int, int>, std::vector<const E4m3Item*>> by;
  for (const E4m3Item& it : l.items) {
    REQUIRE(it.rw == 1 || it.rw == 2 || it.rw == 4, "rw %d", it.rw);
    REQUIRE(it.rows >= 1 && it.rows <= 32 * it.rw && it.rows <= kE4m3Rows, "rows %d", it.rows);
    REQUIRE(it.page_begin >= 0 && it.page_begin < it.page_end, "pages");
    by[{it.table_off, it.kv_head, it.row0}].push_back(&it);
  }
  std::vector<int> part_uses((std::size_t)l.parts, 0);
  std::size_t cut = 0;
  for (const SessionRec& r : st.sessions)
    for (int h = 0; h < st.kv_heads; ++h) {
      const int rows = r.n_new * st.group;
      for (int row0 = 0; row0 < rows;) {
        const auto found = by.find({r.table_off, h, row0});
        REQUIRE(found != by.end(), "row %d of head %d", row0, h);
        std::vector<const E4m3Item*> v = found->second;
        by.erase(found);
        std::sort(v.begin(), v.end(), [](auto* a, auto* b) { return a->page_begin < b->page_begin; });
        int page = 0;
        for (std::size_t k = 0; k < v.size(); ++k) {
          const E4m3Item& it = *v[k];
          REQUIRE(it.page_begin == page, "gap before page %d", it.page_begin);
          page = it.page_end;
          REQUIRE(it.rows == v[0]->rows && it.rw == v[0]->rw && it.ctx == r.ctx && it.q_row == r.q_row, "copies");
          if (v.size() == 1) {
            REQUIRE(it.part == -1, "part of a whole tile");
            continue;
          }
          REQUIRE(it.merge >= 0 && it.merge < (int)l.merges.size() && it.merge == v[0]->merge, "merge");
          const E4m3Merge& m = l.merges[(std::size_t)it.merge];
          REQUIRE(it.part == m.first_part + (int)k && m.n_parts == (int)v.size(), "part %d", it.part);
          REQUIRE(m.rows == it.rows && m.row0 == row0 && m.kv_head == h && m.q_row == r.q_row, "merge record");
          REQUIRE(it.rows <= l.part_rows, "rows of a partial state");
          REQUIRE(it.part < l.parts && part_uses[(std::size_t)it.part]++ == 0, "slot %d twice", it.part);
        }
        cut += v.size() > 1;
        const int last = r.ctx + (row0 + v[0]->rows - 1) / st.group;  // position that the last row sees
        REQUIRE(page == last / 16 + 1, "pages up to %d of position %d", page, last);
        row0 += v[0]->rows;
        REQUIRE(row0 <= rows, "rows");
      }
    }
  REQUIRE(by.empty() && cut == l.merges.size(), "items or merges left");
  for (int u : part_uses) REQUIRE(u == 1, "unused partial slot");
}

}  // namespace

int main(int argc, char** argv) {
  E4m3Lists l;
  std::mt19937 rng(7);
  if (argc == 7) {
    int a[6];
    for (int i = 0; i < 6; ++i) a[i] = std::atoi(argv[i + 1]);
    Desc d;
    for (int i = 0; i < a[5]; ++i) d.add(a[3], a[4], 1, rng);
    const Step st = step_of(d, a[0], a[1], a[2], 1);
    build_e4m3(st, 256, a[2] > 128 ? 1 : a[2] > 64 ? 2 : 3, l);
    check_attention(st, l);
    int longest = 0;
    for (const E4m3Item& it : l.items) longest = std::max(longest, it.page_end - it.page_begin);
    std::printf("items %zu groups %d parts %d rw %d longest %d\n", l.items.size(), l.groups, l.parts, l.items[0].rw,
                longest);
    return 0;
  }
  const int shapes[][3] = {{28, 4, 128}, {14, 2, 64}, {16, 8, 256}, {64, 1, 128}, {5, 5, 8}, {128, 1, 64}, {64, 1, 200}};
  for (int run = 0; run < 400; ++run) {
    const int* sh = shapes[run % 7];
    const int group = sh[0] / sh[1], kind = (int)(rng() % 3), pool = run % 5 == 0 ? 40 : 2000000;
    Desc d;
    for (int i = 1 + (int)(rng() % (kind == 0 ? 60 : 6)); i > 0; --i) {
      const int pick = (int)(rng() % 4);
      const int ctx = pick == 0 ? 0 : pick == 1 ? 16 * (int)(rng() % 200) : (int)(rng() % (pick == 2 ? 200 : 40000));
      const bool few = kind == 0 || (kind == 2 && rng() % 2);
      d.add(ctx, 1 + (int)(rng() % (few ? std::max(1, 64 / group) : 700)), pool, rng);
    }
    const Step st = step_of(d, sh[0], sh[1], sh[2], pool);
    build_e4m3(st, run % 11 == 0 ? 4 : 256, sh[2] > 128 ? 1 : sh[2] > 64 ? 2 : 3, l);
    check_append(st, l);
    check_attention(st, l);
  }
  std::printf("plan_e4m3_check ok\n");
  return 0;
}
