// Planning of a step on an e4m3 pool: see plan_e4m3.hpp.
#include "plan_e4m3.hpp"

#include <algorithm>
#include <utility>

namespace tge::plan {

namespace {

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Rows of one (session, KV head) that meet the same pages, and what they cost
// a workgroup.
struct Tile {
  int session, kv_head, row0, rows, rw, pages;
};

// A piece of a tile: pages [begin, end), the piece `index` of `of`.
struct Piece {
  int tile, begin, end, index, of;
};

using Group = std::vector<Piece>;

// Costs in microseconds of a workgroup while every slot is busy.
struct Costs {
  double page;    // a page
  double start;   // an item's start and end
  double cut;     // a piece of a cut tile: its partial state and share of the merge
  double merge;   // a launch with cut tiles: the last merge
  double solo;    // cost of a page, relative, where the compute unit's other slots are idle
  double uneven;  // what the longest item adds to a launch, relative
  int grain;      // pages that the waves share out at a time
  int least;      // pages of a piece
  int rounds;     // pieces at most, in slots

  // `n` items of `total` in all, the longest of `pages`.
  double time(double total, long long n, int pages, int slots, bool cut) const {
    double t = std::max(total / slots + uneven * (pages * page + start), pages * page * solo + start);
    // (a last round of few items runs faster, but a round it is)
    const long long full = n / slots;
    const double last = (double)n / slots - full;
    if (full > 0) t = std::max(t, total / n * (full + (last == 0.0 ? 0.0 : last <= 0.5 ? 0.6 : 1.0)));
    return t + (cut ? merge : 0.0);
  }
};

// A decode page is bound by HBM (a slot's share of 5.6 TB/s), a prompt page by
// the matrix cores and the exponentials; waves that share their pages (a larger
// rw) pay less for the copies. From launches of 28/4 heads of 128 dims, two
// workgroups a unit (us at rw 1 / 2 / 4: 2048 tokens 56 / 49 / 50, 512 behind
// 1536 24 / 31 / 42, 8192 tokens 567 / 508 / 470, 1333 behind 14003 in shares
// 328 / 318 / 300) a page costs a workgroup 0.15-0.16 / 0.27-0.30 / 0.51-0.58.
// 64-dim blocks, three workgroups a unit, take two thirds of that (32/8 heads,
// 4096 tokens 104 / 92 / 90), 256-dim ones, one a unit, as much (16/8 heads, 1000
// behind 9000 218 / 207 / 199). A cut piece: 4096 tokens of 28/4 heads at rw 4
// uncut 138, in halves 162; at rw 2 143 and 168.
Costs costs_of(int rw, bool prompt, int width, int slots) {
  if (!prompt) return Costs{32.0 * width * slots / 5.6e6, 4.5, 2.0, 4.0, 0.25, 0.05, 8, 40, 1};
  const double page = rw == 1 ? 0.155 : rw == 2 ? 0.285 : 0.53;
  const int grain = rw == 1 ? 8 : 4;
  if (width > 128) return Costs{1.05 * page, 6.0, 6.0 * rw, 6.0 + 2.0 * rw, 1.0, 0.25, grain, 32, 4};
  return Costs{width < 128 ? 0.66 * page : page, 4.0, 3.0 * rw, 4.0 + rw, 0.7, 0.25, grain, 32, 4};
}

// Each tile in equal pieces of at most `len` pages, a piece a group.
std::vector<Group> pieces(const std::vector<Tile>& tiles, int len, const Costs& c) {
  std::vector<Group> groups;
  for (std::size_t i = 0; i < tiles.size(); ++i) {
    const int n = ceil_div(tiles[i].pages, len);
    const int each = ceil_div(ceil_div(tiles[i].pages, n), c.grain) * c.grain, of = ceil_div(tiles[i].pages, each);
    for (int k = 0; k < of; ++k)
      groups.push_back({Piece{(int)i, k * each, std::min((k + 1) * each, tiles[i].pages), k, of}});
  }
  return groups;
}

// Of the piece lengths the one with the least time.
int piece_length(const std::vector<Tile>& tiles, int slots, const Costs& c, double* time) {
  // (tiles of one length count together)
  int most = 0, best = 0;
  for (const Tile& t : tiles) most = std::max(most, t.pages);
  std::vector<int> count((std::size_t)most + 1, 0), lengths;
  for (const Tile& t : tiles)
    if (count[(std::size_t)t.pages]++ == 0) lengths.push_back(t.pages);
  *time = 1e30;
  for (int len = ceil_div(most, c.grain) * c.grain;;) {
    long long n = 0;
    double total = 0.0;
    for (int pages : lengths) {
      const int of = ceil_div(pages, len), k = count[(std::size_t)pages];
      n += (long long)of * k;
      total += k * (pages * c.page + of * c.start + (of > 1 ? of * c.cut : 0.0));
    }
    if (best && n > (long long)slots * c.rounds) break;
    const double t = c.time(total, n, std::min(len, most), slots, len < most);
    if (t < *time) {
      *time = t;
      best = len;
    }
    len = std::min(len - c.grain, len * 15 / 16 / c.grain * c.grain);
    if (len < c.least) break;
  }
  return best;
}

// The tiles end to end, cut into equal shares, a share a group. (Smaller shares
// for the workgroups that land on a compute unit after others, or a part of
// every tile in a queue for those that end first, gained nothing: 64 sessions
// of 1k to 32k tokens, 28/4 heads of 128 dims, 118.8 us; 121.8 with shares 18 %
// apart, 121 with a tenth of the pages queued, 127 with a fifth.)
class Shares {
 public:
  Shares(const std::vector<Tile>& tiles, int slots, const Costs& c) : tiles_(tiles), c_(c) {
    double total = 0.0;
    for (const Tile& t : tiles) total += t.pages * c.page + c.start;
    share_ = std::max(total / slots + 0.5 * c.start, c.least * c.page + c.start);
    auto count = [&](int group, const Tile& t, int begin, int end) {
      cut_pieces += begin > 0 || end < t.pages;
      return group < slots;
    };
    while (!walk(count)) {  // (until the shares are no more than the slots)
      share_ *= 1.01;
      cut_pieces = 0;
    }
    time = share_ + 0.5 * c.start + (cut_pieces ? c.merge : 0.0);
  }

  std::vector<Group> groups() const {
    std::vector<Group> out;
    std::size_t first = 0;  // group of the tile's first piece
    walk([&](int group, const Tile& t, int begin, int end) {
      if (out.size() <= (std::size_t)group) out.emplace_back();
      if (begin == 0) first = (std::size_t)group;
      const int tile = (int)(&t - tiles_.data());
      out.back().push_back(Piece{tile, begin, end, group - (int)first, 1});
      if (end == t.pages)  // a group holds one piece of a tile at most
        for (std::size_t g = first; g < out.size(); ++g)
          (g == first ? out[g].back() : out[g].front()).of = group - (int)first + 1;
      return true;
    });
    return out;
  }

  double time = 0.0;  // (without the cut pieces' own)
  int cut_pieces = 0;

 private:
  // put(group, tile, begin, end) for every piece, until it returns false.
  template <class Put>
  bool walk(Put put) const {
    const int least = std::min(c_.least, 2 * c_.grain);
    double left = 0.0;
    int group = -1;
    for (const Tile& t : tiles_)
      for (int begin = 0; begin < t.pages;) {
        if (left < c_.start + least * c_.page || group < 0) {
          ++group;
          left = share_;
        }
        int n = std::min(t.pages - begin, std::max(least, (int)((left - c_.start) / c_.page) / c_.grain * c_.grain));
        if (t.pages - begin - n < least) n = t.pages - begin;  // (no slivers)
        if (!put(group, t, begin, begin + n)) return false;
        begin += n;
        left -= n * c_.page + c_.start;
      }
    return true;
  }

  const std::vector<Tile>& tiles_;
  Costs c_;
  double share_ = 0.0;
};

// Workgroup b runs on XCD b mod 8, each with an L2 of its own and slots / 8
// workgroups: the pieces of one (session, KV head), which read the same pages,
// go to few XCDs, every XCD gets about the same work, the longest first. (8192
// tokens, 28/4 heads of 128 dims: 782 us with the longest of all heads first on
// every XCD.)
std::vector<Group> by_xcd(const std::vector<Tile>& tiles, std::vector<Group> groups, int slots) {
  constexpr int X = 8;
  const std::size_t n = groups.size();
  std::vector<int> pages(n);
  std::vector<std::size_t> order(n);
  int streams = 0;
  std::vector<int> stream(n);
  for (std::size_t i = 0; i < n; ++i) {
    const Tile& t = tiles[(std::size_t)groups[i][0].tile];
    if (i > 0) {
      const Tile& u = tiles[(std::size_t)groups[i - 1][0].tile];
      streams += t.session != u.session || t.kv_head != u.kv_head;
    }
    stream[i] = streams;
    for (const Piece& p : groups[i]) pages[i] += p.end - p.begin;
    order[i] = i;
  }
  ++streams;
  std::stable_sort(order.begin(), order.end(), [&](std::size_t a, std::size_t b) { return pages[a] > pages[b]; });
  std::vector<std::size_t> list[X];
  long long load[X] = {};
  for (std::size_t i : order) {
    // the stream's own XCDs, then any with room
    const int lo = stream[i] * X / streams, hi = std::max(lo + 1, ((stream[i] + 1) * X + streams - 1) / streams);
    int best = -1;
    for (int x = lo; x < std::min(hi, X); ++x)
      if (list[x].size() < (n - x + X - 1) / X && (best < 0 || load[x] < load[best])) best = x;
    for (int x = 0; best < 0 && x < X; ++x)
      if (list[x].size() < (n - x + X - 1) / X) best = x;
    list[best].push_back(i);
    load[best] += pages[i];
  }
  // Where all groups are resident at once, the second workgroup of a compute
  // unit is short where the first is long.
  for (auto& l : list) {
    const std::size_t half = (std::size_t)slots / (2 * X);
    if (n <= (std::size_t)slots && l.size() > half) std::reverse(l.begin() + (long)half, l.end());
  }
  std::vector<Group> out;
  out.reserve(n);
  for (std::size_t i = 0; i < n; ++i) out.push_back(std::move(groups[list[i % X][i / X]]));
  return out;
}

}  // namespace

void build_e4m3(const Step& s, int cus, int per_cu, E4m3Lists& out) {
  const int slots = cus * per_cu;
  out.tiles.clear();
  out.items.clear();
  out.merges.clear();
  out.groups = out.parts = 0;
  out.part_rows = 32;
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

  // ---- attention. Sessions of up to 64 rows a KV head are one tile each,
  // whose pages nothing else reads.
  const int g = s.group;
  std::vector<Tile> decode;
  bool prompts = false;
  for (std::size_t i = 0; i < s.sessions.size(); ++i) {
    const SessionRec& r = s.sessions[i];
    const int rows = r.n_new * g;
    if (rows > 64) {
      prompts = true;
      continue;
    }
    for (int h = 0; h < s.kv_heads; ++h)
      decode.push_back(Tile{(int)i, h, 0, rows, rows <= 32 ? 1 : 2, ceil_div(r.ctx + r.n_new, 16)});
  }
  auto prompt_tiles = [&](int rw) {
    std::vector<Tile> t;
    for (std::size_t i = 0; i < s.sessions.size(); ++i) {
      const SessionRec& r = s.sessions[i];
      const int rows = r.n_new * g;
      for (int h = 0; rows > 64 && h < s.kv_heads; ++h)
        for (int row0 = 0; row0 < rows; row0 += 32 * rw) {
          const int n = std::min(32 * rw, rows - row0);
          t.push_back(Tile{(int)i, h, row0, n, rw, ceil_div(r.ctx + (row0 + n - 1) / g + 1, 16)});
        }
    }
    return t;
  };

  // A workgroup's first item has its index, its later ones follow the firsts.
  auto add = [&](const std::vector<Tile>& tiles, const std::vector<Group>& groups, bool once) {
    // pieces of a cut tile own consecutive partial slots
    std::vector<int> merge(tiles.size(), -1);
    for (const Group& gr : groups) {
      std::size_t at = (std::size_t)out.groups++;
      for (const Piece& p : gr) {
        const Tile& t = tiles[(std::size_t)p.tile];
        const SessionRec& r = s.sessions[(std::size_t)t.session];
        int& m = merge[(std::size_t)p.tile];
        if (p.of > 1 && m < 0) {
          m = (int)out.merges.size();
          out.part_rows = std::max(out.part_rows, 32 * t.rw);
          out.merges.push_back(E4m3Merge{out.parts, p.of, t.rows, t.row0, t.kv_head, r.q_row, {}});
          out.parts += p.of;
        }
        const int part = p.of > 1 ? out.merges[(std::size_t)m].first_part + p.index : -1;
        if (&p != &gr[0]) {
          out.items[at].next = (int)out.items.size();
          at = out.items.size();
          out.items.emplace_back();
        }
        out.items[at] = E4m3Item{t.kv_head, p.begin, p.end, part, t.row0, t.rows, r.ctx, r.q_row, r.table_off, m,
                                 t.rw, once ? 1 : 0, -1, {}};
      }
    }
  };

  double time = 0.0;
  auto plan_decode = [&](int n, double* t) {
    const Costs c = costs_of(1, false, s.block_dims, slots);
    const int len = piece_length(decode, n, c, t);
    const Shares x(decode, n, c);
    if (*t <= x.time) return pieces(decode, len, c);
    *t = x.time;
    return x.groups();
  };
  auto plan_prompts = [&](int n, std::vector<Tile>* tiles, double* t) {
    std::vector<Group> best;
    *t = 1e30;
    for (int rw : {4, 2, 1}) {
      std::vector<Tile> x = prompt_tiles(rw);
      int shortest = x[0].pages, longest = 0;
      for (const Tile& i : x) {
        shortest = std::min(shortest, i.pages);
        longest = std::max(longest, i.pages);
      }
      if (rw < 4 && best.size() >= 4 * (std::size_t)n) break;  // (large tiles alone fill the device)
      const Costs c = costs_of(rw, true, s.block_dims, slots);
      double e = 0.0;
      const int len = piece_length(x, n, c, &e);
      if (e < *t) {
        *t = e;
        best = pieces(x, len, c);
        *tiles = x;
      }
      // Tiles of like length, too few to even out over the slots, as shares
      // (pieces / shares, us: 28/4 heads of 128 dims, 1333 behind 14003 317 /
      // 300, 1000 behind 30000 462 / 440; 16/8 of 256, 2000 behind 30000 1100 /
      // 1058; not 28/4 of 128, 4096 tokens 139 / 225, 2048 behind 2048 104 /
      // 130, whose tiles' lengths differ; nor 64/8, 2048 behind 8000 572 / 606,
      // two tiles a slot).
      if (2 * shortest < longest || x.size() >= 2 * (std::size_t)n) continue;
      const Shares y(x, n, c);
      if (y.time + c.cut * y.cut_pieces / n < *t) {
        *t = y.time + c.cut * y.cut_pieces / n;
        best = y.groups();
        *tiles = std::move(x);
      }
    }
    return by_xcd(*tiles, std::move(best), n);
  };
  std::vector<Group> dg, pg;
  std::vector<Tile> pt;
  if (!prompts) {
    dg = plan_decode(slots, &time);
  } else if (decode.empty()) {
    pg = plan_prompts(slots, &pt, &time);
  } else {
    // both kinds: slots in proportion to the work
    double d = 0.0, p = 0.0;
    dg = plan_decode(slots, &d);
    pg = plan_prompts(slots, &pt, &p);
    const int n = std::max(1, std::min(slots - 1, (int)(slots * d / (d + p) + 0.5)));
    dg = plan_decode(n, &d);
    pg = plan_prompts(slots - n, &pt, &p);
  }
  out.items.resize(dg.size() + pg.size());
  add(decode, dg, true);
  add(pt, pg, false);
}

}  // namespace tge::plan
