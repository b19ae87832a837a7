// Planning of a step on an e4m3 pool: see plan_e4m3.hpp.
#include "plan_e4m3.hpp"

#include <algorithm>

namespace tge::plan {

namespace {

// Pages a piece of a split tile has at least; a workgroup's start and the
// merge cost about as much as this many pages.
constexpr int kMinPages = 32;
constexpr int kStartPages = 12;

int ceil_div(int a, int b) { return (a + b - 1) / b; }

struct Tile {
  int session, kv_head, row0, rows, rw, pages;
};

}  // namespace

void build_e4m3(const Step& s, int slots, E4m3Lists& out) {
  out.tiles.clear();
  out.items.clear();
  out.wg_first.clear();
  out.merges.clear();
  out.groups = out.parts = 0;
  out.page_twice = false;

  // ---- append: the pages that new rows fall into
  int row = 0;
  for (const SessionRec& r : s.sessions) {
    for (int pos = r.ctx; pos < r.ctx + r.n_new;) {
      const int slot = pos % 16, n = std::min(16 - slot, r.ctx + r.n_new - pos);
      out.tiles.push_back(E4m3Tile{s.tables[(std::size_t)(r.table_off + pos / 16)], row, slot, n, pos, {}});
      row += n;
      pos += n;
    }
  }
  std::vector<char> seen((std::size_t)s.pages, 0);
  for (const E4m3Tile& t : out.tiles) {
    if (seen[(std::size_t)t.page]) out.page_twice = true;
    seen[(std::size_t)t.page] = 1;
  }

  // ---- attention: tiles of rows. Sessions of up to 64 rows a KV head are one
  // tile, whose blocks nothing else reads; longer ones are cut into the
  // largest tiles that still fill the device, since a larger tile reads its
  // pages less often.
  const int g = s.group;
  long long prompt_rows = 0;
  for (const SessionRec& r : s.sessions)
    if (r.n_new * g > 64) prompt_rows += r.n_new * g;
  int prw = 4;
  while (prw > 1 && (prompt_rows * s.kv_heads) / (32 * prw) < slots) prw /= 2;
  std::vector<Tile> once, again;
  for (std::size_t i = 0; i < s.sessions.size(); ++i) {
    const SessionRec& r = s.sessions[i];
    const int rows = r.n_new * g;
    if (rows <= 64) {
      for (int h = 0; h < s.kv_heads; ++h)
        once.push_back(Tile{(int)i, h, 0, rows, rows <= 32 ? 1 : 2, ceil_div(r.ctx + r.n_new, 16)});
      continue;
    }
    for (int row0 = 0; row0 < rows; row0 += 32 * prw) {
      const int n = std::min(32 * prw, rows - row0);
      for (int h = 0; h < s.kv_heads; ++h)
        again.push_back(Tile{(int)i, h, row0, n, prw, ceil_div(r.ctx + (row0 + n - 1) / g + 1, 16)});
    }
  }
  auto emit = [&](const Tile& t, int begin, int end, int part, int merge, int once_flag) {
    const SessionRec& r = s.sessions[(std::size_t)t.session];
    out.items.push_back(E4m3Item{t.kv_head, begin, end, part, t.row0, t.rows, r.ctx, r.q_row, r.table_off, merge,
                                 t.rw, once_flag, {}});
  };
  auto merge_of = [&](const Tile& t, int n) {
    const SessionRec& r = s.sessions[(std::size_t)t.session];
    out.merges.push_back(E4m3Merge{out.parts, n, t.rows, t.row0, t.kv_head, r.q_row, {}});
    out.parts += n;
    return (int)out.merges.size() - 1;
  };

  // Tiles read once: laid end to end and cut into equal shares.
  long long cost = 0;
  for (const Tile& t : once) cost += t.pages + kStartPages;
  const long long share = std::max<long long>(kMinPages + kStartPages, (cost + slots - 1) / slots);
  long long left = 0;  // of the current workgroup's share
  for (const Tile& t : once) {
    // the pieces of this tile: end page, and whether a workgroup starts with the piece
    std::vector<std::pair<int, bool>> cuts;
    for (int at = 0; at < t.pages;) {
      const bool fresh = left < kStartPages + 8;
      if (fresh) left = share;
      int n = (int)std::min<long long>(t.pages - at, left - kStartPages);
      if (n < t.pages - at) n = n / 8 * 8;
      if (t.pages - at - n < 8) n = t.pages - at;  // no slivers
      n = std::min(n, kE4m3ItemPages);
      left -= n + kStartPages;
      at += n;
      cuts.emplace_back(at, fresh);
    }
    const int n = (int)cuts.size(), first = out.parts;
    const int merge = n > 1 ? merge_of(t, n) : -1;
    int at = 0;
    for (int i = 0; i < n; ++i) {
      if (cuts[(std::size_t)i].second) out.wg_first.push_back((int)out.items.size());
      emit(t, at, cuts[(std::size_t)i].first, n > 1 ? first + i : -1, merge, 1);
      at = cuts[(std::size_t)i].first;
    }
  }

  // Prompt tiles: one piece a workgroup, the longest first; pieces of a tile
  // are of equal length, short enough to fill the device.
  if (!again.empty()) {
    long long pages = 0;
    for (const Tile& t : again) pages += t.pages;
    const int most = (int)std::min<long long>(
        kE4m3ItemPages, std::max<long long>(kMinPages, (pages + slots - 1) / slots));
    std::vector<int> cut(again.size());
    const bool fill = (int)again.size() < slots;  // fewer tiles than workgroups
    for (std::size_t i = 0; i < again.size(); ++i)
      cut[i] = ceil_div(again[i].pages, fill ? most : kE4m3ItemPages);
    std::vector<std::size_t> order(again.size());
    for (std::size_t i = 0; i < order.size(); ++i) order[i] = i;
    std::stable_sort(order.begin(), order.end(), [&](std::size_t a, std::size_t b) {
      return ceil_div(again[a].pages, cut[a]) > ceil_div(again[b].pages, cut[b]);
    });
    for (std::size_t i : order) {
      const Tile& t = again[i];
      const int n = cut[i], first = out.parts;
      const int merge = n > 1 ? merge_of(t, n) : -1;
      for (int k = 0; k < n; ++k) {
        out.wg_first.push_back((int)out.items.size());
        emit(t, (int)((long long)t.pages * k / n), (int)((long long)t.pages * (k + 1) / n), n > 1 ? first + k : -1,
             merge, 0);
      }
    }
  }
  out.groups = (int)out.wg_first.size();
  out.wg_first.push_back((int)out.items.size());
}

}  // namespace tge::plan
