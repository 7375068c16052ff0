// Plans of random batches (csrc/batch_plan_build.h), read as the attention
// kernel reads them: every position a row sees lies in exactly one of its items,
// every item and slot inside the plan's room, every cut row block joined once.

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "batch_plan_build.h"

static char last_error[512];
int aegkv_set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(last_error, sizeof last_error, fmt, ap);
  va_end(ap);
  return code;
}
void aegkv_clear_error() { last_error[0] = 0; }

#include "plan.cpp"

using namespace aegkv_batch;

#define REQUIRE(c)                                              \
  do {                                                          \
    if (!(c)) {                                                 \
      printf("line %d: %s (%s)\n", __LINE__, #c, last_error);   \
      exit(1);                                                  \
    }                                                           \
  } while (0)

static std::mt19937 rng(7);
static int64_t below(int64_t n) { return static_cast<int64_t>(rng() % static_cast<uint64_t>(n)); }

struct Made {
  std::vector<int64_t> offsets{0}, ids, lens, fresh;
};

static Made make(int seqs, int64_t longest, int64_t most_new, int bs) {
  Made m;
  int64_t next = 0;
  for (int s = 0; s < seqs; ++s) {
    const int64_t len = below(4) ? 1 + below(longest) : below(3);
    const int64_t fresh = std::min(len, below(5) || len > 400 ? below(most_new + 1) : len);
    const int64_t columns = (len + bs - 1) / bs + below(2);
    for (int64_t c = 0; c < columns; ++c) m.ids.push_back(next++);
    m.offsets.push_back(static_cast<int64_t>(m.ids.size()));
    m.lens.push_back(len);
    m.fresh.push_back(fresh);
  }
  return m;
}

static int plan_of(const Made& m, int64_t blocks, int bs, int kv, int heads, int64_t window,
                   int64_t sinks, const int64_t* room, std::vector<char>* buf, int update) {
  int64_t n = static_cast<int64_t>(buf->size());
  if (!update) {
    const int rc = aegkv_batch_plan(static_cast<int64_t>(m.lens.size()), m.offsets.data(),
                                    m.ids.data(), m.lens.data(), m.fresh.data(), blocks, bs, kv,
                                    heads, window, sinks, room[0], room[1], room[2], 0, nullptr,
                                    &n);
    if (rc) return rc;
    buf->assign(static_cast<size_t>(n), 0x55);
  }
  return aegkv_batch_plan(static_cast<int64_t>(m.lens.size()), m.offsets.data(), m.ids.data(),
                          m.lens.data(), m.fresh.data(), blocks, bs, kv, heads, window, sinks,
                          room[0], room[1], room[2], update, buf->data(), &n);
}

static void check_plan(const Made& m, const std::vector<char>& buf, int bs, int kv, int heads,
                       int64_t window, int64_t sinks) {
  Header h;
  std::memcpy(&h, buf.data(), sizeof h);
  const Room& room = h.room;
  REQUIRE(room.bytes == static_cast<int64_t>(buf.size()));
  REQUIRE(h.num_seqs == static_cast<int32_t>(m.lens.size()) && h.num_seqs <= room.seqs);
  REQUIRE(h.num_tokens <= room.tokens && h.new_spans <= room.new_spans &&
          h.read_spans <= room.read_spans && h.merges <= room.merges);
  std::vector<Seq> seq(m.lens.size());
  if (!seq.empty())
    std::memcpy(seq.data(), buf.data() + room.at_seqs, seq.size() * sizeof(Seq));
  std::vector<int32_t> table(static_cast<size_t>(room.columns));
  if (!table.empty()) std::memcpy(table.data(), buf.data() + room.at_table, table.size() * 4);
  const int group = heads / kv;
  int64_t token = 0, read = 0, news = 0, reads = 0;
  for (size_t s = 0; s < seq.size(); ++s) {
    REQUIRE(seq[s].token == token && seq[s].read_token == read && seq[s].read_span == reads);
    for (int64_t c = 0; c < (m.lens[s] + bs - 1) / bs; ++c)
      REQUIRE(table[seq[s].table + c] == m.ids[m.offsets[s] + c]);
    token += m.fresh[s];
    read += m.lens[s];
    for (int64_t g = 0; g * kSpan < m.lens[s]; ++g) {
      ++reads;
      const int64_t from = std::max(g * kSpan, m.lens[s] - m.fresh[s]);
      const int64_t end = std::min<int64_t>(m.lens[s], (g + 1) * kSpan);
      if (from >= end) continue;
      NewSpan n;
      std::memcpy(&n, buf.data() + room.at_new_spans + news++ * sizeof n, sizeof n);
      REQUIRE(n.block == m.ids[m.offsets[s] + from / bs] && n.inside == from % bs &&
              n.count == end - from && n.inside + n.count <= bs &&
              n.token == seq[s].token + from - (m.lens[s] - m.fresh[s]));
    }
  }
  REQUIRE(news == h.new_spans && reads == h.read_spans && read == h.read_tokens);
  // (kind, seq, kv head, row block) -> tiles of its items
  std::map<std::tuple<int, int, int, int>, std::vector<Item>> found;
  for (int kind = 0; kind < kKinds; ++kind) {
    REQUIRE(h.items[kind] <= room.items[kind] && h.slots[kind] <= room.slots[kind]);
    std::set<int32_t> slots;
    for (int i = 0; i < h.items[kind]; ++i) {
      Item it;
      std::memcpy(&it, buf.data() + room.at_items[kind] + i * sizeof(Item), sizeof it);
      REQUIRE(it.seq >= 0 && it.seq < h.num_seqs && it.kv_head >= 0 && it.kv_head < kv);
      REQUIRE(it.rows > 0 && it.rows <= kKindRows[kind] && it.row % kKindRows[kind] == 0);
      REQUIRE(it.row + it.rows <= m.fresh[it.seq] * group && it.tile < it.tile_end);
      REQUIRE(it.base == m.lens[it.seq] - m.fresh[it.seq] && it.token == seq[it.seq].token &&
              it.table == seq[it.seq].table);
      if (it.slot >= 0) REQUIRE(it.slot < room.slots[kind] && slots.insert(it.slot).second);
      found[{kind, it.seq, it.kv_head, it.row}].push_back(it);
    }
  }
  std::map<std::tuple<int, int, int, int>, Merge> merges;
  std::set<std::tuple<int, int, int, int>> merged;
  for (int i = 0; i < h.merges; ++i) {
    Merge g;
    std::memcpy(&g, buf.data() + room.at_merges + i * sizeof(Merge), sizeof g);
    // every row of a cut block once, found by the block's first
    REQUIRE(g.rows > 0 && g.rows <= (g.parts <= kMergeRows ? kMergeRows : 1));
    for (int32_t r = 0; r < g.rows; ++r)
      REQUIRE(merged.insert({g.kind, g.seq, g.kv_head, g.row + r}).second);
    if (g.first == 0) REQUIRE(merges.insert({{g.kind, g.seq, g.kv_head, g.row}, g}).second);
    REQUIRE((g.row - g.first) % kKindRows[g.kind] == 0);
  }
  size_t cut = 0;
  int64_t rows_found = 0;
  for (const auto& f : found) {
    std::vector<Item> items = f.second;
    std::sort(items.begin(), items.end(),
              [](const Item& x, const Item& y) { return x.tile < y.tile; });
    const Item& a = items[0];
    const int64_t len = m.lens[a.seq], base = len - m.fresh[a.seq];
    rows_found += a.rows;
    std::set<int64_t> tiles;
    for (size_t i = 0; i < items.size(); ++i) {
      REQUIRE(i == 0 || items[i].tile == items[i - 1].tile_end);
      for (int32_t v = items[i].tile; v < items[i].tile_end; ++v) {
        const int64_t t = v < a.first_tiles ? v : v - a.first_tiles + a.window_tile;
        REQUIRE(t >= 0 && t * kTile < len);                  // its first block exists
        REQUIRE(seq[a.seq].table + (t * kTile + kTile - 1) / bs < room.columns);
        REQUIRE((t * kTile + kTile - 1) / bs <= (len + bs - 1) / bs);
        REQUIRE(tiles.insert(t).second);
      }
      REQUIRE((items.size() > 1) == (items[i].slot >= 0));
      if (items.size() > 1) REQUIRE(items[i].slot == items[0].slot + static_cast<int32_t>(i));
    }
    if (items.size() > 1) {
      ++cut;
      const auto g = merges.find(f.first);
      REQUIRE(g != merges.end() && g->second.slot == items[0].slot &&
              g->second.parts == static_cast<int32_t>(items.size()));
      for (int32_t r = 0; r < a.rows; ++r)
        REQUIRE(merged.erase({std::get<0>(f.first), a.seq, a.kv_head, a.row + r}) == 1);
    }
    for (int32_t r : {a.row, a.row + a.rows / 2, a.row + a.rows - 1}) {
      const int64_t p = base + r / group;
      for (int64_t t = 0; t <= p / kTile; ++t) {   // a tile is seen by its ends
        const int64_t low = t * kTile, high = std::min(p, low + kTile - 1);
        if (!window || p - high < window || low < sinks) REQUIRE(tiles.count(t));
      }
    }
  }
  REQUIRE(cut == merges.size() && merged.empty());
  int64_t want_rows = 0;
  for (int64_t f : m.fresh) want_rows += f * group;
  REQUIRE(rows_found == want_rows * kv);
}

// One long sequence among many short ones is cut, however many those are.
static void check_long_among_short() {
  Made m;
  for (int s = 0; s < 3000; ++s) {
    const int64_t len = s == 1234 ? 100000 : 40;
    for (int64_t c = 0; c < (len + 15) / 16; ++c)
      m.ids.push_back(static_cast<int64_t>(m.ids.size()));
    m.offsets.push_back(static_cast<int64_t>(m.ids.size()));
    m.lens.push_back(len);
    m.fresh.push_back(1);
  }
  const int64_t room[3] = {0, 0, 0};
  std::vector<char> buf;
  REQUIRE(plan_of(m, 1 << 20, 16, 4, 16, 0, 0, room, &buf, 0) == 0);
  check_plan(m, buf, 16, 4, 16, 0, 0);
  Header h;
  std::memcpy(&h, buf.data(), sizeof h);
  int32_t longest = 0;
  for (int i = 0; i < h.items[kFew]; ++i) {
    Item it;
    std::memcpy(&it, buf.data() + h.room.at_items[kFew] + i * sizeof(Item), sizeof it);
    longest = std::max(longest, it.tile_end - it.tile);
  }
  REQUIRE(longest <= 400);   // of 3125 tiles
}

int main() {
  check_long_among_short();
  int updates = 0;
  for (int round = 0; round < 400; ++round) {
    const int sizes[] = {16, 32, 64, 128};
    const int bs = sizes[below(4)], kv = 1 + static_cast<int>(below(4));
    const int groups[] = {1, 2, 7, 16, 40};
    const int heads = kv * groups[below(5)];
    const int64_t window = below(2) ? 0 : 1 + below(300), sinks = below(2) ? 0 : below(70);
    const int64_t longest = below(6) ? 400 : 30000;
    const int64_t most_new = below(2) ? 1 : 60;
    Made m = make(static_cast<int>(below(9)), longest, most_new, bs);
    const int64_t blocks = 1 << 20;
    const bool roomy = below(2);
    const int64_t room[3] = {roomy ? 9 : 0, roomy ? 4000 : 0, roomy ? 1200 : 0};
    std::vector<char> buf;
    REQUIRE(plan_of(m, blocks, bs, kv, heads, window, sinks, room, &buf, 0) == 0);
    check_plan(m, buf, bs, kv, heads, window, sinks);
    for (int again = 0; again < 3; ++again) {
      const std::vector<char> was = buf;
      Made next = make(static_cast<int>(below(9)), 400, most_new, bs);
      const int rc = plan_of(next, blocks, bs, kv, heads, window, sinks, room, &buf, 1);
      if (rc == 0) {
        check_plan(next, buf, bs, kv, heads, window, sinks);
        ++updates;
      } else {
        REQUIRE(rc == AEGKV_ENOMEM && buf == was);
      }
    }
  }
  REQUIRE(updates > 300);
  printf("clean\n");
  return 0;
}
