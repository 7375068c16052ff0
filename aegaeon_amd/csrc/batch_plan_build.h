// Building the plan of a batch (batch_plan.h). Host-only; part of plan.cpp.
#ifndef AEGKV_BATCH_PLAN_BUILD_H
#define AEGKV_BATCH_PLAN_BUILD_H

#include "aegkv.h"
#include "batch_plan.h"
#include "errors.h"

#include <algorithm>
#include <cstring>
#include <functional>
#include <queue>
#include <vector>

namespace aegkv_batch {

// Positions are 32-bit in the kernels, with room for a tile behind the last.
constexpr int64_t kMostTokens = (int64_t(1) << 31) - 1024;

// Cutting rows over workgroups. All times are of 4-bit caches; a 16-bit cache takes the same
// cuts, and has not been measured with others. Whole rows, the longest first, where the chip is
// evenly full of them (48 sequences of 40 heads: 119 us cut at every 1/1024 of the
// tiles, 104 whole); else the cut whose estimated time is least. Equal shares of the
// flattened tiles, a workgroup going from one sequence's end to the next one's
// beginning, were slower than items of unequal size with one workgroup each (64
// requests: 72-80 us, 64), and so was one workgroup of 16 waves a head for few short
// sequences (1,025 tokens: 12.6 us, 10.3 cut and joined; 4,096: 25, 10.4).
//
// How many workgroups of a kind the chip holds at once: at 128-wide heads, on all 256
// CUs. A plan serves any width. At 256 the chip holds 512, 256 and 256; cut for that, 64
// decodes took 104 us instead of 109, two contexts of 60,000 tokens 34 instead of 39, and
// prompts and 40 rows the same.
constexpr int64_t kHeld[kKinds] = {768, 512, 512};
// What a workgroup takes before and behind its tiles, and what joining cut rows
// takes, in the time of a tile.
constexpr int64_t kEnds[kKinds] = {8, 8, 8}, kJoin[kKinds] = {8, 8, 8};
// The most items that rows are cut into, beyond one for each.
constexpr int64_t kCuts[kKinds] = {4096, 2048, 2048};

struct Batch {
  int64_t num_seqs;
  const int64_t* offsets;   // columns of sequence s: ids[offsets[s] .. offsets[s + 1])
  const int64_t* ids;
  const int64_t* lens;
  const int64_t* fresh;
};

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t pad16(int64_t x) { return (x + 15) & ~int64_t(15); }
inline long long ll(int64_t x) { return static_cast<long long>(x); }

// First position inside the window of the earliest of the sequence's queries.
inline int64_t window_begin(const Header& h, int64_t first_query) {
  return h.window ? std::max<int64_t>(0, first_query - h.window + 1) : 0;
}

// Rows [row, row + rows) of a sequence under each KV head, and their tiles.
struct Rows {
  int32_t seq, row, rows;
  int32_t first_tiles, window_tile, tiles;
};

inline int kind_of(int64_t rows) {
  return rows <= kKindRows[kFew] ? kFew : rows <= kMostMore ? kMore : kMany;
}

inline void rows_of(const Header& h, const Batch& b, std::vector<Rows>* out) {
  for (int64_t s = 0; s < b.num_seqs; ++s) {
    const int64_t rows = b.fresh[s] * h.group;
    if (!rows) continue;
    const int kind = kind_of(rows);
    for (int64_t row = 0; row < rows; row += kKindRows[kind]) {
      const int64_t n = std::min<int64_t>(kKindRows[kind], rows - row);
      const int64_t base = b.lens[s] - b.fresh[s];
      const int64_t low = base + row / h.group, high = base + (row + n - 1) / h.group;
      const int64_t window_tile = window_begin(h, low) / kTile;
      const int64_t first_tiles = h.window ? std::min(up(h.sinks, kTile), window_tile) : 0;
      Rows r;
      r.seq = static_cast<int32_t>(s);
      r.row = static_cast<int32_t>(row);
      r.rows = static_cast<int32_t>(n);
      r.first_tiles = static_cast<int32_t>(first_tiles);
      r.window_tile = static_cast<int32_t>(window_tile);
      r.tiles = static_cast<int32_t>(first_tiles + high / kTile + 1 - window_tile);
      out[kind].push_back(r);
    }
  }
}

// The time when every row block's tiles are cut into equal parts of at most
// `each`, and the next of the workgroups that the chip holds takes the longest
// one left. The KV heads are alike: one of them, on its share of the chip,
// stands for all.
inline int64_t time_of(const std::vector<Rows>& rows, int64_t kv_heads, int kind, int64_t each) {
  std::vector<int64_t> sizes;
  bool cut = false;
  for (const Rows& r : rows) {
    const int64_t parts = up(r.tiles, each);
    cut |= parts > 1;
    sizes.insert(sizes.end(), static_cast<size_t>(parts), up(r.tiles, parts) + kEnds[kind]);
  }
  std::sort(sizes.begin(), sizes.end(), std::greater<int64_t>());
  const int64_t copies = std::max<int64_t>(1, kv_heads / kHeld[kind]);
  const size_t held = static_cast<size_t>(std::max<int64_t>(1, kHeld[kind] / kv_heads));
  std::priority_queue<int64_t, std::vector<int64_t>, std::greater<int64_t>> busy;
  int64_t end = 0;
  for (int64_t t : sizes) {
    int64_t from = 0;
    if (busy.size() >= held) {
      from = busy.top();
      busy.pop();
    }
    busy.push(from + t * copies);
    end = std::max(end, from + t * copies);
  }
  return end + (cut ? kJoin[kind] : 0);
}

inline int64_t items_of(const std::vector<Rows>& rows, int64_t kv_heads, int64_t each) {
  int64_t n = 0;
  for (const Rows& r : rows) n += up(r.tiles, each);
  return n * kv_heads;
}

// Tiles of an item at most: of cuts into 1/1 .. 1/8 of what a workgroup would
// take of equal shares, and none at all, the one whose time is least.
inline int64_t share_out(const std::vector<Rows>& rows, int64_t kv_heads, int kind,
                         int64_t most_items) {
  int64_t total = 0, longest = 1;
  for (const Rows& r : rows) {
    total += r.tiles * kv_heads;
    longest = std::max<int64_t>(longest, r.tiles);
  }
  const int64_t count = static_cast<int64_t>(rows.size()) * kv_heads;
  if (count >= 8 * kHeld[kind] && longest * kHeld[kind] <= total) return longest;
  int64_t best = longest, least = time_of(rows, kv_heads, kind, longest);
  for (int64_t eighths = 8; eighths >= 1; --eighths) {
    const int64_t each = std::max<int64_t>(4, up(total * eighths, 8 * kHeld[kind]));
    if (each >= longest) continue;
    const int64_t items = items_of(rows, kv_heads, each);
    if (items > most_items || items > count + kCuts[kind]) break;
    const int64_t t = time_of(rows, kv_heads, kind, each);
    if (t < least) {
      least = t;
      best = each;
    }
    if (each == 4) break;
  }
  return best;
}

// Slots that cuts into items of at most `each` tiles take, and the merges that join them.
struct Parts {
  int64_t slots, merges;
};

inline int64_t merges_of(int64_t rows, int64_t parts) {
  return parts == 1 ? 0 : up(rows, parts <= kMergeRows ? kMergeRows : 1);
}

inline Parts parts_of(const std::vector<Rows>& rows, int64_t kv_heads, int64_t each) {
  Parts p{0, 0};
  for (const Rows& r : rows) {
    const int64_t parts = up(r.tiles, each);
    if (parts > 1) p.slots += parts * kv_heads;
    p.merges += merges_of(r.rows, parts) * kv_heads;
  }
  return p;
}

// Columns of a sequence that its queries see: [0, firsts) and [rest, end), whole blocks.
struct SeenColumns {
  int64_t firsts, rest, end;
};

inline SeenColumns seen_columns(const Header& h, int64_t len, int64_t fresh) {
  if (!fresh) return SeenColumns{0, 0, 0};
  const int64_t begin = window_begin(h, len - fresh);
  const int64_t rest = begin / h.block_size;
  const int64_t firsts = h.window ? std::min<int64_t>(h.sinks, begin) : 0;
  return SeenColumns{std::min(up(firsts, h.block_size), rest), rest, up(len, h.block_size)};
}

inline int check(const Header& h, const Batch& b) {
  std::vector<int64_t> written;   // (block, first, end) of every block written
  int64_t columns = 0, tokens = 0, all = 0;
  for (int64_t s = 0; s < b.num_seqs; ++s) {
    const int64_t len = b.lens[s], fresh = b.fresh[s];
    if (len < 0 || len > kMostTokens)
      return aegkv_set_error(AEGKV_EINVAL, "sequence %lld: length %lld outside [0, %lld]", ll(s),
                             ll(len), ll(kMostTokens));
    if (fresh < 0 || fresh > len)
      return aegkv_set_error(AEGKV_EINVAL, "sequence %lld: %lld new tokens of %lld", ll(s),
                             ll(fresh), ll(len));
    const int64_t lo = b.offsets[s], hi = b.offsets[s + 1];
    if (lo < 0 || hi < lo || (s == 0 && lo != 0))
      return aegkv_set_error(AEGKV_EINVAL, "sequence %lld: bad column offsets", ll(s));
    const int64_t need = up(len, h.block_size);
    if (hi - lo < need)
      return aegkv_set_error(AEGKV_ERANGE, "sequence %lld: %lld tokens in %lld blocks of %d", ll(s),
                             ll(len), ll(hi - lo), h.block_size);
    // (each look at the columns is without branches: a decode step pays them all)
    const int64_t* const ids = b.ids + lo;
    uint64_t outside = 0;       // its sign: that of id + 1 and num_blocks - 1 - id
    for (int64_t c = 0; c < hi - lo; ++c) {
      const uint64_t id = static_cast<uint64_t>(ids[c]);
      outside |= (id + 1) | (static_cast<uint64_t>(h.num_blocks) - 1 - id);
    }
    if (static_cast<int64_t>(outside) < 0)
      for (int64_t c = 0; c < hi - lo; ++c)
        if (ids[c] < -1 || ids[c] >= h.num_blocks)
          return aegkv_set_error(AEGKV_ERANGE, "sequence %lld: block id %lld outside [0, %lld)",
                                 ll(s), ll(ids[c]), ll(h.num_blocks));
    if (fresh) {
      const SeenColumns seen = seen_columns(h, len, fresh);
      int64_t released = 0;     // negative: some
      for (int64_t c = 0; c < seen.firsts; ++c) released |= ids[c];
      for (int64_t c = seen.rest; c < seen.end; ++c) released |= ids[c];
      if (released < 0)
        for (int64_t c = 0; c < need; ++c)
          if (ids[c] < 0 && (c < seen.firsts || c >= seen.rest))
            return aegkv_set_error(AEGKV_ERANGE,
                                   "sequence %lld: column %lld is released but its tokens are "
                                   "seen", ll(s), ll(c));
      for (int64_t c = (len - fresh) / h.block_size; c < need; ++c) {
        const int64_t at = c * h.block_size;
        written.push_back(ids[c]);
        written.push_back(std::max<int64_t>(0, len - fresh - at));
        written.push_back(std::min<int64_t>(h.block_size, len - at));
      }
    }
    columns += need + 1;
    tokens += fresh;
    all += need;
  }
  if (columns > kMostTokens || tokens > kMostTokens / std::max(1, h.heads) ||
      all > kMostTokens / (h.block_size / kSpan))
    return aegkv_set_error(AEGKV_ENOMEM, "a batch of %lld columns and %lld new tokens is too large",
                           ll(columns), ll(tokens));
  std::vector<size_t> order(written.size() / 3);
  for (size_t i = 0; i < order.size(); ++i) order[i] = i;
  std::sort(order.begin(), order.end(), [&](size_t x, size_t y) {
    return std::make_pair(written[3 * x], written[3 * x + 1]) <
           std::make_pair(written[3 * y], written[3 * y + 1]);
  });
  for (size_t i = 1; i < order.size(); ++i) {
    const int64_t* a = &written[3 * order[i - 1]];
    const int64_t* c = &written[3 * order[i]];
    if (a[0] == c[0] && c[1] < a[2])
      return aegkv_set_error(AEGKV_EDUP, "token %lld of block %lld is written twice", ll(c[1]),
                             ll(c[0]));
  }
  return 0;
}

// Whether some block is in two places that queries see: sequences without new tokens, and
// columns before a window, gather no weights.
inline bool shares(const Header& h, const Batch& b, int64_t columns) {
  const auto each = [&](const auto& f) {
    for (int64_t s = 0; s < b.num_seqs; ++s) {
      const int64_t* const ids = b.ids + b.offsets[s];
      const SeenColumns seen = seen_columns(h, b.lens[s], b.fresh[s]);
      for (int64_t c = 0; c < seen.firsts; ++c) f(ids[c]);
      for (int64_t c = seen.rest; c < seen.end; ++c) f(ids[c]);
    }
  };
  if (h.num_blocks / 64 <= columns + 1024) {
    std::vector<uint64_t> seen(static_cast<size_t>(h.num_blocks / 64 + 1));
    uint64_t twice = 0;
    each([&](int64_t id) {
      uint64_t& word = seen[static_cast<size_t>(id >> 6)];
      const uint64_t bit = uint64_t(1) << (id & 63);
      twice |= word & bit;
      word |= bit;
    });
    return twice != 0;
  }
  // few columns of very many blocks
  std::vector<int64_t> all;
  each([&](int64_t id) { all.push_back(id); });
  std::sort(all.begin(), all.end());
  return std::adjacent_find(all.begin(), all.end()) != all.end();
}

// What of the plan depends on the sequences, into a buffer with room for it.
inline int fill(Header& h, const Batch& b, const std::vector<Rows>* rows, char* base) {
  const Room& room = h.room;
  auto* seq = reinterpret_cast<Seq*>(base + room.at_seqs);
  auto* table = reinterpret_cast<int32_t*>(base + room.at_table);
  auto* merge = reinterpret_cast<Merge*>(base + room.at_merges);
  auto* span = reinterpret_cast<NewSpan*>(base + room.at_new_spans);
  auto* tile = reinterpret_cast<PlaceTile*>(base + room.at_place_tiles);
  int64_t columns = 0, tokens = 0, new_spans = 0, read_spans = 0, read_tokens = 0;
  int64_t place_tiles = 0;
  h.complete = 1;
  for (int64_t s = 0; s < b.num_seqs; ++s) columns += up(b.lens[s], h.block_size) + 1;
  for (int64_t s = 0; s < b.num_seqs; ++s) tokens += b.fresh[s];
  if (b.num_seqs > room.seqs || columns > room.columns || tokens > room.tokens)
    return aegkv_set_error(AEGKV_ENOMEM, "%lld sequences, %lld columns and %lld new tokens do not "
                           "fit a plan of %lld, %lld and %lld", ll(b.num_seqs), ll(columns),
                           ll(tokens), ll(room.seqs), ll(room.columns), ll(room.tokens));
  h.shared = shares(h, b, columns);
  columns = tokens = 0;
  for (int64_t s = 0; s < b.num_seqs; ++s) {
    const int64_t len = b.lens[s], fresh = b.fresh[s], need = up(len, h.block_size);
    seq[s].len = static_cast<int32_t>(len);
    seq[s].fresh = static_cast<int32_t>(fresh);
    seq[s].table = static_cast<int32_t>(columns);
    seq[s].token = static_cast<int32_t>(tokens);
    seq[s].read_span = static_cast<int32_t>(read_spans);
    seq[s].pad = 0;
    seq[s].read_token = read_tokens;
    const int64_t* const ids = b.ids + b.offsets[s];
    int32_t* const to = table + columns;
    int64_t released = 0;       // negative: some
    for (int64_t c = 0; c < need; ++c) {
      released |= ids[c];
      const int32_t id = static_cast<int32_t>(ids[c]);
      to[c] = id & ~(id >> 31);     // 0 for -1
    }
    if (released < 0) h.complete = 0;
    table[columns + need] = 0;   // the tile behind the last block may look here
    columns += need + 1;
    tokens += fresh;
    for (int64_t at = len - fresh; at < len;) {
      const int64_t end = std::min(len, (at / kSpan + 1) * kSpan);
      if (new_spans >= room.new_spans)
        return aegkv_set_error(AEGKV_ENOMEM, "the new tokens do not fit the plan's %lld spans",
                               ll(room.new_spans));
      span[new_spans++] = NewSpan{table[seq[s].table + at / h.block_size],
                                  static_cast<uint16_t>(at % h.block_size),
                                  static_cast<uint16_t>(end - at),
                                  static_cast<int32_t>(seq[s].token + at - (len - fresh)),
                                  static_cast<int32_t>(at)};
      at = end;
    }
    read_spans += up(len, kSpan);
    read_tokens += len;
  }
  h.num_seqs = static_cast<int32_t>(b.num_seqs);
  h.num_tokens = static_cast<int32_t>(tokens);
  h.new_spans = static_cast<int32_t>(new_spans);
  h.read_spans = static_cast<int32_t>(read_spans);
  const int64_t window = h.window ? h.window : INT32_MAX;
  for (const bool many : {true, false}) {
    for (int64_t s = 0; s < b.num_seqs; ++s) {
      const int64_t len = b.lens[s], fresh = b.fresh[s], base = len - fresh;
      if (fresh == 0 || (fresh * h.group > kMostMore) != many) continue;
      for (int64_t at = 0; at < len; at += kPlaceTile) {
        if (base - (at + kPlaceTile - 1) >= window && at >= h.sinks) continue;
        if (place_tiles >= room.place_tiles)
          return aegkv_set_error(AEGKV_ENOMEM, "the sequences do not fit the plan's %lld tiles of "
                                 "places", ll(room.place_tiles));
        tile[place_tiles++] = PlaceTile{static_cast<int32_t>(s), static_cast<int32_t>(at)};
      }
    }
    if (many) h.many_tiles = static_cast<int32_t>(place_tiles);
  }
  h.place_tiles = static_cast<int32_t>(place_tiles);
  h.read_tokens = read_tokens;
  if (read_spans > room.read_spans)
    return aegkv_set_error(AEGKV_ENOMEM, "%lld spans to read do not fit the plan", ll(read_spans));
  int64_t merges = 0;
  for (int kind = 0; kind < kKinds; ++kind) {
    const std::vector<Rows>& all = rows[kind];
    if (static_cast<int64_t>(all.size()) * h.kv_heads > room.items[kind])
      return aegkv_set_error(AEGKV_ENOMEM, "the plan has no room for sequences of this many new "
                             "tokens (%s rows under a KV head)",
                             kind == kMany ? "over 64" : kind == kMore ? "17 to 64" : "up to 16");
    int64_t each = share_out(all, h.kv_heads, kind, room.items[kind]);
    // a plan that was cut to another batch may have room for fewer parts: whole rows
    // need none
    for (Parts p = parts_of(all, h.kv_heads, each);
         p.slots > room.slots[kind] || merges + p.merges > room.merges;
         p = parts_of(all, h.kv_heads, each))
      each *= 2;
    // the longest go first, so that the last to end are short
    std::vector<size_t> order(all.size());
    for (size_t i = 0; i < order.size(); ++i) order[i] = i;
    const auto size = [&](size_t i) { return up(all[i].tiles, up(all[i].tiles, each)); };
    std::stable_sort(order.begin(), order.end(),
                     [&](size_t x, size_t y) { return size(x) > size(y); });
    auto* item = reinterpret_cast<Item*>(base + room.at_items[kind]);
    int64_t items = 0, slots = 0;
    for (size_t i : order) {
      const Rows& r = all[i];
      const int64_t parts = up(r.tiles, each);
      for (int32_t head = 0; head < h.kv_heads; ++head) {
        const int64_t slot = slots;
        for (int64_t p = 0; p < parts; ++p)
          item[items++] = Item{r.seq, head, r.row, r.rows,
                               static_cast<int32_t>(r.tiles * p / parts),
                               static_cast<int32_t>(r.tiles * (p + 1) / parts), r.first_tiles,
                               r.window_tile, parts > 1 ? static_cast<int32_t>(slots++) : -1,
                               seq[r.seq].len - seq[r.seq].fresh, seq[r.seq].token,
                               seq[r.seq].table};
        if (parts == 1) continue;
        const int32_t rows_each = parts <= kMergeRows ? kMergeRows : 1;
        for (int32_t first = 0; first < r.rows; first += rows_each) {
          merge[merges++] = Merge{r.seq, head, r.row + first,
                                  std::min(rows_each, r.rows - first),
                                  static_cast<int32_t>(slot), static_cast<int32_t>(parts), kind,
                                  seq[r.seq].token, first, {0, 0, 0}};
        }
      }
    }
    h.items[kind] = static_cast<int32_t>(items);
    h.slots[kind] = static_cast<int32_t>(slots);
  }
  h.merges = static_cast<int32_t>(merges);
  return 0;
}

// Room for the batch itself, or if bounds are given, for any within them: also where
// this one is as large as they are, as the step is that a graph is captured on.
inline void make_room(Header& h, const Batch& b, const std::vector<Rows>* rows, int64_t max_seqs,
                      int64_t max_columns, int64_t max_tokens) {
  Room& r = h.room;
  int64_t columns = 0, tokens = 0, new_spans = 0, read_spans = 0;
  for (int64_t s = 0; s < b.num_seqs; ++s) {
    const int64_t len = b.lens[s], fresh = b.fresh[s];
    columns += up(len, h.block_size);
    tokens += fresh;
    if (fresh) new_spans += up(len, kSpan) - (len - fresh) / kSpan;
    read_spans += up(len, kSpan);
  }
  const bool exact = max_seqs == 0 && max_columns == 0 && max_tokens == 0;
  r.seqs = std::max(max_seqs, b.num_seqs);
  max_columns = std::max(max_columns, columns);
  r.columns = max_columns + r.seqs;
  r.tokens = std::max(max_tokens, tokens);
  r.new_spans = exact ? new_spans : std::min(r.tokens, r.tokens / kSpan + 2 * r.seqs);
  r.read_spans = exact ? read_spans : max_columns * (h.block_size / kSpan);
  // (a sequence's last tile may hold one place; also where there is room for nothing
  // else, an update may have other lengths in as many blocks)
  r.place_tiles = std::min(max_columns, max_columns * h.block_size / kPlaceTile + r.seqs);
  r.merges = 0;
  int64_t at = pad16(sizeof(Header));
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += pad16(bytes);
    return here;
  };
  r.at_seqs = take(r.seqs * static_cast<int64_t>(sizeof(Seq)));
  r.at_table = take(r.columns * 4);
  r.at_new_spans = take(r.new_spans * static_cast<int64_t>(sizeof(NewSpan)));
  for (int kind = 0; kind < kKinds; ++kind) {
    const int64_t count = static_cast<int64_t>(rows[kind].size()) * h.kv_heads;
    r.items[kind] = r.slots[kind] = 0;
    if (count && exact) {
      const int64_t each = share_out(rows[kind], h.kv_heads, kind, INT32_MAX);
      r.items[kind] = items_of(rows[kind], h.kv_heads, each);
      const Parts p = parts_of(rows[kind], h.kv_heads, each);
      r.slots[kind] = p.slots;
      r.merges += p.merges;
    } else if (count) {
      const int64_t most = (kind == kMany   ? r.tokens * h.group / kManyRows + r.seqs
                            : kind == kMore ? r.seqs * (kMostMore / kKindRows[kMore])
                                            : r.seqs) *
                           h.kv_heads;
      r.items[kind] = most + kCuts[kind];
      // row by row where one has more than kMergeRows parts
      const int64_t many = std::min(most, r.items[kind] / (kMergeRows + 1));
      r.slots[kind] = r.items[kind];
      r.merges += most * up(kKindRows[kind], kMergeRows) + many * kKindRows[kind];
    }
    r.at_items[kind] = take(r.items[kind] * static_cast<int64_t>(sizeof(Item)));
  }
  r.at_merges = take(r.merges * static_cast<int64_t>(sizeof(Merge)));
  r.at_place_tiles = take(r.place_tiles * static_cast<int64_t>(sizeof(PlaceTile)));
  r.bytes = at;
}

inline int describe(Header& h, int64_t num_blocks, int32_t block_size, int32_t kv_heads,
                    int32_t heads, int64_t window, int64_t sinks) {
  std::memset(&h, 0, sizeof h);
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128)
    return aegkv_set_error(AEGKV_EINVAL, "a block holds 16, 32, 64 or 128 tokens, not %d",
                           block_size);
  if (num_blocks <= 0 || num_blocks > INT32_MAX)
    return aegkv_set_error(AEGKV_EINVAL, "%lld blocks outside [1, 2^31)", ll(num_blocks));
  if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || heads > 65535)
    return aegkv_set_error(AEGKV_EINVAL, "%d query heads over %d KV heads", heads, kv_heads);
  if (window < 0 || sinks < 0)
    return aegkv_set_error(AEGKV_EINVAL, "window %lld and sinks %lld must not be negative",
                           ll(window), ll(sinks));
  h.magic = kMagic;
  h.num_blocks = num_blocks;
  h.block_size = block_size;
  h.kv_heads = kv_heads;
  h.heads = heads;
  h.group = heads / kv_heads;
  h.window = window > kMostTokens ? 0 : static_cast<int32_t>(window);
  h.sinks = static_cast<int32_t>(std::min(sinks, kMostTokens));
  return 0;
}

}  // namespace aegkv_batch

#endif  // AEGKV_BATCH_PLAN_BUILD_H
