// Whether rows of values share a byte (csrc/value_places.h), against every byte
// looked at.

#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "value_places.h"

using namespace aegkv_batch;

#define REQUIRE(c)                               \
  do {                                           \
    if (!(c)) {                                  \
      printf("line %d: %s\n", __LINE__, #c);     \
      exit(1);                                   \
    }                                            \
  } while (0)

static const char* at(int64_t i) { return reinterpret_cast<const char*>(uintptr_t(1) << 20) + i; }

static std::vector<char> bytes_of(const Place& p) {
  std::vector<char> held(4096, 0);
  for (int64_t t = 0; t < p.tokens; ++t)
    for (int64_t h = 0; h < p.heads; ++h)
      for (int64_t b = 0; b < p.run; ++b)
        held[static_cast<size_t>(p.begin - (uintptr_t(1) << 20) + t * p.token + h * p.head + b)] = 1;
  return held;
}

static bool share(const Place& a, const Place& b) {
  const std::vector<char> x = bytes_of(a), y = bytes_of(b);
  for (size_t i = 0; i < x.size(); ++i)
    if (x[i] && y[i]) return true;
  return false;
}

int main() {
  std::mt19937 rng(3);
  const auto below = [&](int64_t n) { return static_cast<int64_t>(rng() % uint64_t(n)); };
  int apart = 0, shared = 0;
  for (int round = 0; round < 200000; ++round) {
    const int64_t tokens = below(6), heads = 1 + below(5), run = 1 + below(9);
    const int64_t token = below(4) ? run * heads + below(60) : below(12);
    const int64_t head = below(4) ? run + below(12) : below(80);
    const Place a = place(at(below(200)), tokens, heads, run, token, head);
    const Place b = place(at(below(200)), tokens, heads, run, token, head);
    // alike but for their beginnings: exactly
    REQUIRE(overlap(a, b) == share(a, b));
    REQUIRE(overlap(a, b) == overlap(b, a));
    (share(a, b) ? shared : apart) += 1;
    REQUIRE(!tokens || overlap(a, a));
    REQUIRE(same(a, a) && same(a, b) == (a.begin == b.begin));
    // unlike: never missed, and apart where their ranges are
    const Place c = below(2) ? place(at(below(400)), below(90))
                             : place(at(below(400)), below(5), 1 + below(5), 1 + below(9),
                                     below(60), below(60));
    if (share(a, c)) REQUIRE(overlap(a, c) && overlap(c, a));
    int64_t first[2], last[2];
    const Place* both[2] = {&a, &c};
    for (int i = 0; i < 2; ++i) {
      const std::vector<char> held = bytes_of(*both[i]);
      first[i] = 5000;
      last[i] = -1;
      for (int64_t k = 0; k < 4096; ++k)
        if (held[static_cast<size_t>(k)]) first[i] = std::min(first[i], k), last[i] = k;
    }
    if (last[0] < first[1] || last[1] < first[0]) REQUIRE(!overlap(a, c) && !overlap(c, a));
  }
  REQUIRE(apart > 20000 && shared > 20000);
  // sizes as they come: one V beside K in a fused projection, and in place
  const int64_t big = int64_t(1) << 33;
  const Place q = place(at(0), 1 << 20, 32, 256, big / 1024, 256);
  REQUIRE(!overlap(q, place(at(8192), 1 << 20, 32, 256, big / 1024, 256)));
  REQUIRE(overlap(q, place(at(8191), 1 << 20, 32, 256, big / 1024, 256)));
  REQUIRE(overlap(q, place(at(big / 1024), 1 << 20, 32, 256, big / 1024, 256)));
  printf("clean\n");
  return 0;
}
