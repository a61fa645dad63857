// Division of the attention of rows that share leading pages (csrc/kernels/prefix_attn.cu and beside it; ops/prefix.py keeps the
// result): which rows share what, ranges of keys, units for the blocks.
//
// A batch that changes is planned anew before its next pass, so that this is a part of what a pass costs.
#include <algorithm>
#include <cstdint>
#include <cstring>
#include <vector>

namespace {

constexpr int kUnit = 8;                       // numbers of a unit: slot, first row, rows, first key, end key, part, tail, head

// Mirrors ops/prefix.py PlanShape.  Times in us.
struct Shape {
  int rows, heads, kv_heads, vdim, page_tokens, chunk, rows_per_unit, together, grid, min_tokens, max_turns, max_units, max_cells, extra;
  int least_span, reserved;                    // keys that a range is a multiple of
  double turn, row, longer, shorter, byte, part;
};

struct Group {
  int begin, end, pages;                       // of the sorted rows
};

int leased(const int32_t* row, int width) {
  int n = 0;
  while (n < width && row[n] >= 0) ++n;
  return n;
}

// Sorts rows [begin, end) of `order`, which agree before column `col`, by the columns from there on; shares[i]: leased pages that sorted
// rows i and i + 1 have in common.
void sort_rows(const int32_t* table, int width, std::vector<int>& order, std::vector<int>& shares, int begin, int end, int col) {
  if (end - begin < 2) return;
  const int32_t* lead = table + 1ll * order[begin] * width;
  int differ = width;
  for (int i = begin + 1; i < end; ++i) {
    const int32_t* row = table + 1ll * order[i] * width;
    int c = col;
    while (c < differ && row[c] == lead[c] && lead[c] >= 0) ++c;
    differ = c;
  }
  if (differ == width || lead[differ] < 0) {   // none of them goes on, or the first one does not: find out which
    bool same = true;
    if (differ < width)
      for (int i = begin + 1; i < end && same; ++i) same = table[1ll * order[i] * width + differ] < 0;
    if (same) {
      for (int i = begin; i + 1 < end; ++i) shares[i] = differ;
      return;
    }
  }
  auto at = [&](int row) { return std::max(table[1ll * row * width + differ], -1); };
  std::stable_sort(order.begin() + begin, order.begin() + end, [&](int a, int b) { return at(a) < at(b); });
  for (int i = begin; i < end;) {
    int j = i + 1;
    while (j < end && at(order[j]) == at(order[i])) ++j;
    if (at(order[i]) < 0)
      for (int k = i; k + 1 < j; ++k) shares[k] = differ;
    else
      sort_rows(table, width, order, shares, i, j, differ + 1);
    if (j < end) shares[j - 1] = differ;
    i = j;
  }
}

// Groups of rows that begin with the same leased pages, a row in one group at most.  A range of the sorted rows shares the least of the
// runs between neighbours; the range that saves most reads, (rows - 1) x pages, is a group, and the rows on either side are divided again.
void find_groups(const int32_t* table, int n, int width, std::vector<int>& order, std::vector<Group>& groups) {
  order.resize(n);
  for (int i = 0; i < n; ++i) order[i] = i;
  std::vector<int> shares(n > 0 ? n : 1, 0);
  sort_rows(table, width, order, shares, 0, n, 0);
  struct Best {
    long long gain;
    int pages, begin, end;
    bool operator<(const Best& o) const {
      return gain != o.gain ? gain < o.gain : pages != o.pages ? pages < o.pages : begin != o.begin ? begin < o.begin : end < o.end;
    }
  };
  std::vector<std::pair<int, int>> todo{{0, std::max(n - 1, 0)}}, rising;      // rising: (first run, height) of the ranges still open
  while (!todo.empty()) {
    const auto [lo, hi] = todo.back();
    todo.pop_back();
    Best best{0, 0, 0, 0};
    rising.clear();
    for (int i = lo; i <= hi; ++i) {
      const int h = i < hi ? shares[i] : 0;
      int from = i;
      while (!rising.empty() && rising.back().second >= h) {
        from = rising.back().first;
        const int top = rising.back().second;
        rising.pop_back();
        best = std::max(best, Best{1ll * (i - from) * top, top, from, i});
      }
      rising.push_back({from, h});
    }
    if (best.gain == 0) continue;
    groups.push_back({best.begin, best.end + 1, best.pages});
    todo.push_back({lo, std::max(lo, best.begin - 1)});
    todo.push_back({std::min(hi, best.end + 1), hi});
  }
}

struct Shared {
  int begin, rows, pieces, slot;               // rows: order[begin] ..
  int low, tokens;                             // keys [low, tokens)
};
struct Tail {
  int first, rows, slot, key0;
  int keys;                                    // there are now
  int group;                                   // its rows' prefix, -1: none
};
struct Item {
  int slot, first, rows, key0, key1, part, tail;
  int keys;                                    // that it has now
};
// A block as one number that compares as (time that it is busy, turns, block): the time in tenths of a nanosecond.
using Block = uint64_t;
constexpr int kTurnBits = 20, kIdBits = 8;
Block block(double busy, int turns, int id) {
  return (static_cast<uint64_t>(busy * 1e4) << kTurnBits | static_cast<uint64_t>(turns)) << kIdBits | static_cast<uint64_t>(id);
}

class Division {
 public:
  Division(const Shape& s, const std::vector<Shared>& shared, const std::vector<Tail>& tails, int rows, int limit)
      : s_(s), shared_(shared), tails_(tails), rows_(rows), limit_(limit) {}

  // The best division found; its time, or -1: none.
  struct Plan {
    double time = -1;
    int span = 0;
    std::vector<Item> items;                   // the longest first
    std::vector<int> ranks, place, parts;      // ranks: groups of items by time; place: of (rank, head)
  } best;

  // Lengths that the keys may be divided by, by the time that they take at least: every one that may be shorter is tried.
  void search() {
    static const int spans[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 28, 32, 40, 48, 64, 96, 128, 192, 256, 384, 512, 1024, 2048, 4096};
    long long longest = 0, room = static_cast<long long>(tails_.size()) + s_.extra;
    for (const Shared& x : shared_) {
      longest = std::max<long long>(longest, x.tokens - x.low);
      room += x.pieces;
    }
    for (const Tail& t : tails_) longest = std::max<long long>(longest, t.keys);
    const long long unit = s_.least_span;
    std::vector<std::pair<double, long long>> tries;
    for (int k : spans)
      if (k * unit < longest) bound(k * unit, room, tries);
    bound((longest + unit - 1) / unit * unit, room, tries);           // divides nothing
    std::sort(tries.begin(), tries.end());
    for (const auto& [least, span] : tries)
      if (best.time < 0 || least < best.time) attempt(span);
  }

 private:
  const Shape& s_;
  const std::vector<Shared>& shared_;
  const std::vector<Tail>& tails_;
  const int rows_, limit_;
  Plan now_;
  std::vector<double> need_;
  std::vector<Block> blocks_;

  double join_time(long long parts, int most) const { return 8.0 * parts * s_.heads * s_.vdim * s_.byte + most * s_.part; }

  void bound(long long span, long long room, std::vector<std::pair<double, long long>>& tries) const {
    long long items = 0, keys = 0, parts = 0, most = 0, longest = 0, second = 0;
    auto item = [&](long long length, long long count) {
      if (length > longest) {
        second = count > 1 ? length : longest;
        longest = length;
      } else if (length > second || (length == longest && count > 0)) {
        second = length;
      }
    };
    for (const Shared& x : shared_) {
      const long long n = (x.tokens - x.low + span - 1) / span;
      items += x.pieces * n;
      keys += 1ll * x.pieces * (x.tokens - x.low);
      parts += x.rows * n;
      item(std::min<long long>(span, x.tokens - x.low), x.pieces * std::max(1ll, (x.tokens - x.low) / span));
    }
    for (const Tail& t : tails_) {
      const long long n = std::max(1ll, t.keys / span);
      items += n;
      keys += t.keys;
      parts += t.rows * n;
      item(t.keys - (n - 1) * span, 1);
      most = std::max(most, n + (t.group >= 0 ? (shared_[t.group].tokens - shared_[t.group].low + span - 1) / span : 0));
    }
    if (items > room) return;
    const double at_a_time = 1.0 * s_.grid * s_.together / s_.kv_heads;
    const double per_key = s_.together == 1 ? s_.longer : (s_.longer + s_.shorter) / 2;
    const double busy = (items * s_.turn + parts * s_.row + keys * per_key) / at_a_time;
    const double last = s_.turn + s_.row + s_.longer * longest + (s_.together > 1 ? s_.shorter * second : 0);      // the first block's first turn
    tries.push_back({std::max(busy, last) + join_time(parts, static_cast<int>(most)), span});
  }

  void attempt(long long span) {
    std::vector<Item>& items = now_.items;
    items.clear();
    now_.parts.assign(rows_, 0);
    for (const Shared& x : shared_) {
      const int n = static_cast<int>((x.tokens - x.low + span - 1) / span);
      for (int i = 0; i < x.pieces; ++i) {
        const int lo = static_cast<int>(1ll * x.rows * i / x.pieces), hi = static_cast<int>(1ll * x.rows * (i + 1) / x.pieces);
        for (int k = 0; k < n; ++k) {
          const int key0 = static_cast<int>(x.low + k * span), key1 = static_cast<int>(std::min<long long>(x.tokens, x.low + (k + 1) * span));
          items.push_back({x.slot, x.begin + lo, hi - lo, key0, key1, k, 0, key1 - key0});
        }
      }
    }
    shared_parts(span);
    for (const Tail& t : tails_) {
      const int n = static_cast<int>(std::max(1ll, t.keys / span)), part = now_.parts[t.first];
      for (int k = 0; k < n; ++k) {            // the last one goes on to wherever the request gets
        const int key0 = static_cast<int>(t.key0 + k * span), key1 = k + 1 < n ? static_cast<int>(key0 + span) : limit_;
        items.push_back({t.slot, t.first, t.rows, key0, key1, part + k, 1, std::min(key1 - key0, std::max(1, t.key0 + t.keys - key0))});
      }
      for (int r = 0; r < t.rows; ++r) now_.parts[t.first + r] += n;
    }
    // those that a block has at a time side by side: pieces that walk the same keys, if there are two
    std::sort(items.begin(), items.end(), [](const Item& a, const Item& b) {
      return a.keys != b.keys ? a.keys > b.keys : a.slot != b.slot ? a.slot < b.slot : a.key0 != b.key0 ? a.key0 < b.key0 : a.first < b.first;
    });
    const int w = s_.together, n = static_cast<int>(items.size()), groups = (n + w - 1) / w;
    need_.resize(groups);
    for (int g = 0; g < groups; ++g) {
      int most = 0, longest = 0, sum = 0;
      for (int i = g * w; i < std::min(n, (g + 1) * w); ++i) {
        most = std::max(most, items[i].rows);
        longest = std::max(longest, items[i].keys);
        sum += items[i].keys;
      }
      need_[g] = s_.turn + s_.row * most + s_.longer * longest + s_.shorter * (sum - longest);
    }
    now_.ranks.resize(groups);
    for (int g = 0; g < groups; ++g) now_.ranks[g] = g;
    std::stable_sort(now_.ranks.begin(), now_.ranks.end(), [this](int a, int b) { return need_[a] > need_[b]; });
    long long parts = 0;
    int most = 0;
    for (int p : now_.parts) {
      parts += p;
      most = std::max(most, p);
    }
    now_.span = static_cast<int>(span);
    const double join = join_time(parts, most);
    double busy = 0;
    for (double x : need_) busy += x;
    if (best.time >= 0 && std::max(busy * s_.kv_heads / s_.grid, need_[now_.ranks[0]]) + join >= best.time) return;
    now_.time = join + deal(groups);
    if (best.time < 0 || now_.time < best.time) std::swap(best, now_);
  }

  void shared_parts(long long span) {
    for (const Shared& x : shared_)
      for (int i = 0; i < x.rows; ++i) now_.parts[order_[x.begin + i]] = static_cast<int>((x.tokens - x.low + span - 1) / span);
  }

  // Groups to blocks, the longest first, each to the block that has least to do: block b takes the places b, b + grid, b + 2 grid ...
  // Returns the time until the last block is done.
  double deal(int groups) {
    const int total = groups * s_.kv_heads, grid = s_.grid, heads = s_.kv_heads;
    now_.place.resize(total);
    double last = need_[now_.ranks[0]];
    const int first = std::min(grid, total);
    for (int i = 0; i < first; ++i) now_.place[i] = i;
    if (total <= grid) return last;
    blocks_.resize(grid);
    for (int i = 0; i < grid; ++i) blocks_[i] = block(need_[now_.ranks[i / heads]], 1, i);
    std::sort(blocks_.begin(), blocks_.end());          // a heap, too: the least first
    Block latest = blocks_.back();
    int size = grid;
    for (int i = grid; i < total; ++i) {
      Block b = blocks_[0];
      const int id = static_cast<int>(b & ((1 << kIdBits) - 1)), turns = static_cast<int>(b >> kIdBits & ((1 << kTurnBits) - 1));
      now_.place[i] = turns * grid + id;
      b += block(need_[now_.ranks[i / heads]], 1, 0);
      latest = std::max(latest, b);
      if (turns + 1 >= s_.max_turns) b = blocks_[--size];
      int at = 0;
      for (int next = 1; next < size; next = 2 * at + 1) {
        next += next + 1 < size && blocks_[next + 1] < blocks_[next];
        if (blocks_[next] >= b) break;
        blocks_[at] = blocks_[next];
        at = next;
      }
      blocks_[at] = b;
    }
    last = std::max(last, static_cast<double>(latest >> (kTurnBits + kIdBits)) * 1e-4);
    return last;
  }

 public:
  std::vector<int> order_;                     // rows by prefix
};

int divide(const void* shape, const int32_t* table, int slots, int width, const int64_t* row_slot, int n, const int64_t* lengths,
           int used, int32_t* data, const int32_t* at, int32_t* groups, int32_t* result) {
  const Shape& s = *static_cast<const Shape*>(shape);
  const int P = s.page_tokens, limit = width * P;
  if (s.grid > 1 << kIdBits || s.max_turns > 1 << kTurnBits) return -1;
  std::vector<int> index(slots, -1), keep, rows_of, first_of, begin(n, 0), group(n, -1);
  for (int r = 0; r < n; ++r)
    if (row_slot[r] >= 0 && index[row_slot[r]] < 0) {
      index[row_slot[r]] = static_cast<int>(keep.size());
      keep.push_back(static_cast<int>(row_slot[r]));
    }
  const int m = static_cast<int>(keep.size());
  first_of.assign(m + 1, 0);                             // rows of slot keep[i]: rows_of[first_of[i]] ..
  for (int r = 0; r < n; ++r)
    if (row_slot[r] >= 0) ++first_of[index[row_slot[r]] + 1];
  for (int i = 0; i < m; ++i) first_of[i + 1] += first_of[i];
  rows_of.resize(first_of[m]);
  {
    std::vector<int> to(first_of.begin(), first_of.end() - 1);
    for (int r = 0; r < n; ++r)
      if (row_slot[r] >= 0) rows_of[to[index[row_slot[r]]]++] = r;
  }
  auto length = [&](int r) { return static_cast<int>(std::min<int64_t>(std::max<int64_t>(lengths[r], 0), limit)); };
  if (s.chunk > 0 && lengths != nullptr)
    for (int r = 0; r < n; ++r) begin[r] = std::max(length(r) - 1, 0) / s.chunk * s.chunk / P * P;

  // prefixes, of rows that see some of them, from more than one slot
  std::vector<Shared> shared;
  std::vector<int> order, sorted;
  if (m > 1) {
    std::vector<int32_t> own(1ll * m * width);
    for (int i = 0; i < m; ++i) std::memcpy(&own[1ll * i * width], table + 1ll * keep[i] * width, 4ll * width);
    std::vector<Group> found;
    find_groups(own.data(), m, width, sorted, found);
    std::vector<int> rows;
    for (const Group& g : found) {
      const int tokens = g.pages * P;
      int low = tokens, members = 0;
      rows.clear();
      for (int i = g.begin; i < g.end; ++i) {
        const int k = sorted[i];
        bool any = false;
        for (int j = first_of[k]; j < first_of[k + 1]; ++j)
          if (begin[rows_of[j]] < tokens) {
            rows.push_back(rows_of[j]);
            low = std::min(low, begin[rows_of[j]]);
            any = true;
          }
        members += any;
      }
      if (members < 2 || tokens - low < s.min_tokens) continue;
      std::sort(rows.begin(), rows.end());
      const int count = static_cast<int>(rows.size());
      for (int r : rows) {
        group[r] = static_cast<int>(shared.size());
        begin[r] = tokens;
      }
      shared.push_back({static_cast<int>(order.size()), count, (count + s.rows_per_unit - 1) / s.rows_per_unit,
                        static_cast<int>(row_slot[rows[0]]), low, tokens});
      order.insert(order.end(), rows.begin(), rows.end());
    }
  }
  // what is left of every row: neighbours of one slot together, as many as a unit takes
  std::vector<Tail> tails;
  for (int i = 0; i < m; ++i) {
    const int have = lengths == nullptr ? P * leased(table + 1ll * keep[i] * width, width) : 0;
    for (int j = first_of[i]; j < first_of[i + 1];) {
      const int r = rows_of[j];
      int count = 1, longest = lengths == nullptr ? have : length(r);
      while (j + count < first_of[i + 1] && count < s.rows_per_unit && rows_of[j + count] == r + count && begin[r + count] == begin[r] &&
             group[r + count] == group[r]) {
        if (lengths != nullptr) longest = std::max(longest, length(r + count));
        ++count;
      }
      tails.push_back({r, count, keep[i], begin[r], std::max(1, longest - begin[r]), group[r]});
      j += count;
    }
  }

  Division d(s, shared, tails, n, limit);
  d.order_ = order;
  int places = 0;
  std::memset(data + at[1], 0, 4ll * (at[4] + s.rows - at[1]));
  int32_t *turns = data + at[1], *row_order = data + at[2], *cell = data + at[3], *owner = cell + s.rows, *parts = data + at[4];
  if (!tails.empty()) {
    d.search();
    const int total = static_cast<int>(d.best.place.size()), w = s.together;
    int most = 0;
    for (int i = 0; i < total; ++i) most = std::max(most, ++turns[d.best.place[i] % s.grid]);
    places = most * s.grid * w;
    long long cells = 0;
    for (int r = 0; r < n; ++r) cells += d.best.parts[r];
    if (places > s.max_units || cells > s.max_cells) return -1;
    std::memset(data + at[0], 0, 4ll * kUnit * std::max(places, used));
    for (int i = 0; i < total; ++i) {
      const int g = d.best.ranks[i / s.kv_heads];
      for (int e = 0; e < w && g * w + e < static_cast<int>(d.best.items.size()); ++e) {
        const Item& x = d.best.items[g * w + e];
        const int32_t unit[kUnit] = {x.slot, x.first, x.rows, x.key0, x.key1, x.part, x.tail, i % s.kv_heads};
        std::memcpy(data + at[0] + (1ll * d.best.place[i] * w + e) * kUnit, unit, sizeof(unit));
      }
    }
    int sum = 0;
    for (int r = 0; r < n; ++r) {
      cell[r] = sum;
      parts[r] = d.best.parts[r];
      owner[r] = row_slot[r] < 0 ? 0 : static_cast<int32_t>(row_slot[r]) + 1;
      sum += d.best.parts[r];
    }
    for (int r = n; r < s.rows; ++r) cell[r] = sum;
    std::copy(order.begin(), order.end(), row_order);
  } else {
    std::memset(data + at[0], 0, 4ll * kUnit * used);
  }
  data[0] = places;
  data[1] = data[2] = data[3] = 0;
  std::copy(order.begin(), order.end(), groups + 3 * shared.size());
  for (size_t i = 0; i < shared.size(); ++i) {
    groups[3 * i] = shared[i].rows;
    groups[3 * i + 1] = shared[i].tokens;
    groups[3 * i + 2] = shared[i].low;
  }
  result[0] = places;
  result[1] = tails.empty() ? 0 : d.best.span;
  result[2] = static_cast<int>(shared.size());
  return 0;
}

}  // namespace

extern "C" {

// Groups of rows of a page table [n][width] that begin with the same leased pages: rows order[bounds[2 i]] .. order[bounds[2 i + 1] - 1]
// share pages[i].  Returns how many groups there are (n / 2 at most).
int ds41_prefix_groups(const int32_t* table, int n, int width, int32_t* order, int32_t* bounds, int32_t* pages) try {
  std::vector<int> rows;
  std::vector<Group> groups;
  find_groups(table, n, width, rows, groups);
  std::copy(rows.begin(), rows.end(), order);
  for (size_t i = 0; i < groups.size(); ++i) {
    bounds[2 * i] = groups[i].begin;
    bounds[2 * i + 1] = groups[i].end;
    pages[i] = groups[i].pages;
  }
  return static_cast<int>(groups.size());
} catch (...) {
  return -2;
}

// The plan of `n` rows of slots row_slot[] (negative: none) over the page table [slots][width]; `lengths`: tokens of each row's request
// (null: what its pages hold).  `data`: [4 | units | turns | order | cell, owner | parts], the parts at at[0] .. at[4]; units of the
// `used` places that the last plan had and this one has not become zeros.  groups[3 i]: rows of prefix i, its tokens, the first of them
// that any of its rows sees, behind the last prefix all their rows; result: places, length of the ranges, prefixes.
// 0; -1: the plan's arrays do not hold the division; -2: no memory.
int ds41_prefix_divide(const void* shape, const int32_t* table, int slots, int width, const int64_t* row_slot, int n, const int64_t* lengths,
                       int used, int32_t* data, const int32_t* at, int32_t* groups, int32_t* result) try {
  return divide(shape, table, slots, width, row_slot, n, lengths, used, data, at, groups, result);
} catch (...) {
  return -2;
}

}  // extern "C"
