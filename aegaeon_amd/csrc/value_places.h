// Where the values of a call over a paged cache lie, and whether two of them
// share a byte. Host-only; internal to the library.
#ifndef AEGKV_VALUE_PLACES_H
#define AEGKV_VALUE_PLACES_H

#include <algorithm>
#include <cstdint>

namespace aegkv_batch {

// `tokens` times `heads` runs of `run` bytes, `token` and `head` bytes apart (an axis
// of length 1 is 0 apart). tokens 0: nothing.
struct Place {
  uintptr_t begin;
  int64_t tokens, heads, run, token, head;
};

inline Place place(const void* base, int64_t bytes) {
  return Place{reinterpret_cast<uintptr_t>(base), bytes > 0 ? 1 : 0, 1, bytes, 0, 0};
}

inline Place place(const void* base, int64_t tokens, int64_t heads, int64_t run, int64_t token,
                   int64_t head) {
  return Place{reinterpret_cast<uintptr_t>(base), tokens, heads, run, tokens > 1 ? token : 0,
               heads > 1 ? head : 0};
}

inline bool same(const Place& a, const Place& b) {
  return a.begin == b.begin && a.tokens == b.tokens && a.heads == b.heads && a.run == b.run &&
         a.token == b.token && a.head == b.head;
}

// Whether two places share a byte: exactly where they differ in nothing but their
// beginning (slices of one buffer, also interleaved ones), by the range from first to
// last byte of each token where those lie equally far apart, else of the whole.
inline bool overlap(const Place& a, const Place& b) {
  if (!a.tokens || !b.tokens) return false;
  const auto end = [](const Place& p) {
    return p.begin + static_cast<uintptr_t>((p.tokens - 1) * p.token + (p.heads - 1) * p.head +
                                            p.run);
  };
  if (a.begin >= end(b) || b.begin >= end(a)) return false;
  if (!same(a, Place{a.begin, b.tokens, b.heads, b.run, b.token, b.head})) {
    if (!a.token || a.token != b.token) return true;
    // tokens of one length (Q, K and V of a fused projection): by each token's range
    const int64_t apart = static_cast<int64_t>(b.begin - a.begin), next = -apart / a.token;
    for (const int64_t near : {next - 1, next, next + 1}) {
      const int64_t gap = apart + std::clamp(near, 1 - a.tokens, b.tokens - 1) * a.token;
      if (gap < (a.heads - 1) * a.head + a.run && -gap < (b.heads - 1) * b.head + b.run)
        return true;
    }
    return false;
  }
  // runs i tokens and j heads apart for some |i| < tokens, |j| < heads
  const int64_t apart = static_cast<int64_t>(b.begin - a.begin);
  for (int64_t j = 1 - a.heads; j < a.heads; ++j) {
    const int64_t rest = apart - j * a.head;
    const int64_t i = a.token ? rest / a.token : 0;   // the nearest is this or a neighbour
    for (const int64_t near : {i - 1, i, i + 1}) {
      const int64_t n = std::clamp(near, 1 - a.tokens, a.tokens - 1);
      const int64_t gap = rest - n * a.token;
      if (gap < a.run && -gap < a.run) return true;
    }
  }
  return false;
}

}  // namespace aegkv_batch

#endif  // AEGKV_VALUE_PLACES_H
