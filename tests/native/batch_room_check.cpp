// Updates within the room that a plan was made with are taken, whatever batch it
// was made for: also one that fills the room, as a decode step does before capture.

#define main batch_plan_main
#include "batch_plan_check.cpp"
#undef main

static Made of(const std::vector<int64_t>& lens, const std::vector<int64_t>& fresh, int bs) {
  Made m;
  m.lens = lens;
  m.fresh = fresh;
  for (int64_t len : lens) {
    for (int64_t c = 0; c < (len + bs - 1) / bs; ++c)
      m.ids.push_back(static_cast<int64_t>(m.ids.size()));
    m.offsets.push_back(static_cast<int64_t>(m.ids.size()));
  }
  return m;
}

static int64_t total(const std::vector<int64_t>& x) {
  int64_t n = 0;
  for (int64_t i : x) n += i;
  return n;
}

// A batch of up to `seqs` sequences, `columns` columns and `tokens` new tokens with as
// many rows a sequence as some of `kinds` (none new: always).
static Made within(int64_t seqs, int64_t columns, int64_t tokens, const std::set<int>& kinds,
                   int group, int bs) {
  std::vector<int64_t> lens, fresh;
  const int64_t most = below(3) ? seqs : 1 + below(std::max<int64_t>(seqs, 1));
  for (int64_t s = 0; s < std::min(seqs, most); ++s) {
    const int64_t left = most - s;      // long ones too, while there is room
    const int64_t held = below(4) ? std::min(columns, 1 + below(std::max<int64_t>(1, 2 * columns / left)))
                                  : below(columns + 1);
    const int64_t len = held * bs - (held ? below(bs) : 0);
    int64_t f = 0;
    for (int tries = 0; tries < 8 && !f; ++tries) {
      const int64_t up_to = std::min({len, tokens, below(3) ? int64_t(1) : tokens});
      const int64_t some = up_to > 0 ? 1 + below(up_to) : 0;
      if (some && kinds.count(kind_of(some * group))) f = some;
    }
    columns -= held;
    tokens -= f;
    lens.push_back(len);
    fresh.push_back(f);
  }
  return of(lens, fresh, bs);
}

static std::set<int> kinds_of(const Made& m, int group) {
  std::set<int> k;
  for (int64_t f : m.fresh)
    if (f) k.insert(kind_of(f * group));
  return k;
}

static void take(const char* what, const Made& first, const int64_t* room, const Made& next, int bs,
                 int kv, int heads) {
  std::vector<char> buf;
  REQUIRE(plan_of(first, 1 << 22, bs, kv, heads, 0, 0, room, &buf, 0) == 0);
  check_plan(first, buf, bs, kv, heads, 0, 0);
  if (plan_of(next, 1 << 22, bs, kv, heads, 0, 0, room, &buf, 1) != 0) {
    printf("%s: %s\n", what, last_error);
    exit(1);
  }
  check_plan(next, buf, bs, kv, heads, 0, 0);
}

int main() {
  const int64_t a[3] = {64, 6400, 64}, b[3] = {1, 2, 2}, c[3] = {4, 28, 4}, d[3] = {2, 4, 32};
  take("64 to 2", of(std::vector<int64_t>(64, 1600), std::vector<int64_t>(64, 1), 16), a,
       of({1600, 1600}, {1, 1}, 16), 16, 8, 32);
  take("across a block", of({20}, {2}, 16), b, of({17}, {2}, 16), 16, 8, 32);
  take("4 to 1", of({100, 100, 100, 100}, {1, 1, 1, 1}, 16), c, of({448}, {1}, 16), 16, 8, 32);
  take("other places", of({32, 32}, {16, 16}, 16), d, of({31, 32}, {16, 16}, 16), 16, 8, 32);
  // one that was cut to its batch takes a smaller one uncut
  const int64_t none[3] = {0, 0, 0};
  take("no room asked", of({40000}, {1}, 16), none, of({39000}, {1}, 16), 16, 1, 1);
  take("fewer cuts", of({3000, 3000}, {1, 1}, 16), none, of({6000}, {1}, 16), 16, 8, 32);
  for (int round = 0; round < 200; ++round) {
    const int sizes[] = {16, 32, 64, 128};
    const int bs = sizes[below(4)];
    const int kvs[] = {1, 2, 8, 40};
    const int kv = kvs[below(4)];
    const int groups[] = {1, 4, 7, 16};
    const int group = kv == 40 ? 1 : groups[below(4)];
    const int64_t window = below(2) ? 0 : 1 + below(300), sinks = below(2) ? 0 : below(70);
    std::set<int> any{kFew, kMore, kMany};
    const int64_t columns = below(5) ? 20 + below(200) : 2000;
    const Made first = within(1 + below(12), columns, 1 + below(below(2) ? 400 : 12), any, group, bs);
    const std::set<int> kinds = kinds_of(first, group);
    int64_t own = 0;
    for (int64_t len : first.lens) own += (len + bs - 1) / bs;
    // what the batch holds itself, or some more of it
    const int64_t room[3] = {static_cast<int64_t>(first.lens.size()) + (below(3) ? 0 : below(9)),
                             own + (below(3) ? 0 : below(3000)),
                             total(first.fresh) + (below(3) ? 0 : below(500))};
    std::vector<char> buf;
    REQUIRE(plan_of(first, 1 << 22, bs, kv, kv * group, window, sinks, room, &buf, 0) == 0);
    check_plan(first, buf, bs, kv, kv * group, window, sinks);
    for (int again = 0; again < 4; ++again) {
      const Made next = within(room[0], room[1], room[2], kinds, group, bs);
      REQUIRE(plan_of(next, 1 << 22, bs, kv, kv * group, window, sinks, room, &buf, 1) == 0);
      check_plan(next, buf, bs, kv, kv * group, window, sinks);
    }
  }
  printf("clean\n");
  return 0;
}
