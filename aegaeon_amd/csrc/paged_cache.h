// An ordinary paged KV cache (bfloat16 or float16) and rotary positions: kernels
// that rotate rows and write them into the cache, attend over it, add up the
// attention that its tokens gather, and drop those that gathered least. Part of
// aegkv.hip's translation unit; contracts are in include/aegkv.h.
//
// A page holds block_size tokens of kv_heads heads, [token][head][value] or
// [head][token][value]; a block's bytes lie together, blocks any distance apart.
#ifndef AEGKV_PAGED_CACHE_H
#define AEGKV_PAGED_CACHE_H

#include "cache_kernels.h"

namespace {

struct Pages {
  const char* k;
  const char* v;
  int64_t k_block, v_block;   // bytes from one block to the next
  int32_t token, head;        // bytes inside a page
};

// x / by for 0 <= x: a division in 32 bits takes some thirty instructions. `part` is
// 2^32 / by rounded down (by > 1), so the product is the quotient or one less.
struct Divisor {
  uint32_t by, part;
};

__host__ __device__ __forceinline__ Divisor divisor(int32_t by) {
  return Divisor{static_cast<uint32_t>(by),
                 by > 1 ? static_cast<uint32_t>((uint64_t(1) << 32) / static_cast<uint32_t>(by))
                        : 0u};
}

__device__ __forceinline__ int32_t quotient(int32_t x, Divisor d) {
  if (d.by == 1) return x;
  const uint32_t u = static_cast<uint32_t>(x), q = __umulhi(u, d.part);
  return static_cast<int32_t>(q + (u - q * d.by >= d.by));
}

// ---------------------------------------------------------- rotate, write --

// A kind of heads: q, k or v. Where a plan's k and v go is a page; `to` is where else.
struct HeadKind {
  Values from, to;
  const char* pages;          // null: `to`
  int64_t block;              // bytes from one of its blocks to the next
  int32_t heads, turned;      // turned: rotated
  // A workgroup takes `each` heads of up to `chunk` tokens; `groups` of them take all heads,
  // `parts` a span of the plan's. `begin`: the first workgroup of this kind.
  int32_t each, chunk, groups, parts;
  int64_t begin;
};

struct PlaceArgs {
  const char* plan;           // null: tokens are rows, one after another
  int64_t at_new_spans;
  int64_t tokens;             // without a plan
  const double* turns;        // a position's turns, for each pair
  const void* positions;      // null: the plan's
  int32_t position_bytes;
  int32_t pairs, interleaved;
  float amplitude;
  int32_t head_dim;
  HeadKind kinds[3];          // q, k, v
  int32_t page_token, page_head;    // bytes inside a page
  Divisor units, by_pairs;    // items of a head; pairs
};

constexpr int kPlaceLanes = 256;
constexpr int kMostAngles = 2048;   // of a workgroup: 16 tokens of 128 pairs, fewer of more

typedef const AEGKV_CONSTANT char* ArgBytes;

// N values (1, 4 or 8) of 16 or 32 bits as they lie in memory, up to 16 bytes.
template <int N, typename T>
struct Raw {
  static constexpr int kWords = N * sizeof(T) / 4;    // 0: one value of 16 bits
  uint32_t w[kWords ? kWords : 1];

  __device__ __forceinline__ void load(const void* from, bool whole_words, bool whole_lines) {
    if constexpr (kWords > 1) {
      typedef unsigned int words __attribute__((ext_vector_type(kWords)));
      if (whole_words) {
        const auto* p = reinterpret_cast<const words*>(from);
        const words x = whole_lines ? __builtin_nontemporal_load(p) : *p;
        __builtin_memcpy(w, &x, sizeof w);
        return;
      }
    }
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = static_cast<const T*>(from)[i];
    __builtin_memcpy(w, t, sizeof t);
  }
  __device__ __forceinline__ void store(void* to, bool whole_words, bool whole_lines) const {
    if constexpr (kWords > 1) {
      typedef unsigned int words __attribute__((ext_vector_type(kWords)));
      if (whole_words) {
        words x;
        __builtin_memcpy(&x, w, sizeof w);
        auto* p = reinterpret_cast<words*>(to);
        if (whole_lines) __builtin_nontemporal_store(x, p);
        else *p = x;
        return;
      }
    }
    T t[N];
    __builtin_memcpy(t, w, sizeof t);
#pragma unroll
    for (int i = 0; i < N; ++i) static_cast<T*>(to)[i] = t[i];
  }
  __device__ __forceinline__ void widen(float* x) const {
    T t[N];
    __builtin_memcpy(t, w, sizeof t);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = static_cast<float>(t[i]);
  }
  __device__ __forceinline__ void round(const float* x) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = static_cast<T>(x[i]);
    __builtin_memcpy(w, t, sizeof t);
  }
};

__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float x = a * c - b * s;
  b = b * c + a * s;
  a = x;
}

// (a, b) -> (a c - b s, b c + a s) for each pair, c and s the cosine and sine of
// position * turns: the angle in 64 bits, of which the whole turns are dropped before
// it is rounded (positions of millions keep their angle), values in 32, one
// rounding at the end. A workgroup takes a few tokens of some heads of a kind: the angles,
// 150 instructions each, are made once for all of them, while the first values are on
// their way. Bound by HBM, then by its instructions: 12,300 tokens of 3 x 40 heads are
// written in 213 us from float32 (5.1 TB/s) and in 156 from 16 bits (5.2); 16,000 tokens of
// 32 heads are rotated in 47 to 55 us (4.8-5.6 TB/s: the less, the less of them the cache
// behind the L2 still holds), in float32 in 105 (5.0).
// G: type of k and v; T: of q, of what is written and of what comes of q. A lane takes
// two runs of N values of a head at once, half of the rotated part (or of the others) apart:
// both sides of N pairs, or neighbouring pairs in each run where they are interleaved, and
// lanes side by side reach for neighbouring bytes either way. N: 8, 4 for values in
// 32 bits (16 bytes a load), 1 for parts that are no whole runs.
template <int N, typename G, typename T>
__global__ __launch_bounds__(kPlaceLanes) void place_rows_kernel(PlaceArgs a) {
  __shared__ float cosine[kMostAngles], sine[kMostAngles];
  const int kind = blockIdx.x < a.kinds[1].begin ? 0 : blockIdx.x < a.kinds[2].begin ? 1 : 2;
  // read where they are: one of three, by number, would be copied to memory of the lanes'
  const auto* own = reinterpret_cast<const AEGKV_CONSTANT PlaceArgs*>(
                        (ArgBytes)__builtin_amdgcn_kernarg_segment_ptr())->kinds + kind;
  const int32_t index = static_cast<int32_t>(blockIdx.x - own->begin);
  const int32_t run = index / own->groups, first_head = (index - run * own->groups) * own->each;
  const int32_t chunk = own->chunk, heads = min(own->each, own->heads - first_head);
  const bool query = kind == 0, turned = own->turned;
  const int32_t span = run / own->parts, part = (run - span * own->parts) * chunk;
  int64_t token;
  int32_t count, position = 0, block = 0, inside = 0;
  if (a.plan) {
    if (span >= in_plan<Header>(a.plan, 0)->new_spans) return;
    const auto* s = in_plan<NewSpan>(a.plan, a.at_new_spans) + span;
    token = int64_t(s->token) + part;
    count = min(chunk, s->count - part);
    position = s->position + part;
    block = s->block;
    inside = s->inside + part;
    if (count <= 0) return;
  } else {
    token = int64_t(span) * chunk;
    count = static_cast<int32_t>(min<int64_t>(chunk, a.tokens - token));
  }
  const int32_t units = static_cast<int32_t>(a.units.by), items = count * heads * units;
  const bool words = own->from.whole_words;
  // Whole lines go past the caches. Where a head's runs are halves of lines, 16,000 tokens
  // of 32 heads took 68 us that way, 50 through them (three sets of rows in turn).
  const int64_t size = query ? sizeof(T) : sizeof(G);
  const int32_t rest = turned ? a.pairs : 0;      // the part behind the rotated one
  const auto in_lines = [&](int64_t each) {
    return rest * each % 128 == 0 && (a.head_dim / 2 - rest) * each % 128 == 0;
  };
  const bool lines = in_lines(size), to_lines = in_lines(sizeof(T));

  // From and to, of the first token and head; strides in bytes.
  const char* const from = own->from.base + (token * own->from.token +
                                             first_head * own->from.head) * size;
  const int64_t from_token = own->from.token * size, from_head = own->from.head * size;
  const bool paged = own->pages != nullptr, to_words = paged || own->to.whole_words;
  const int64_t to_token = paged ? a.page_token : own->to.token * int64_t(sizeof(T));
  const int64_t to_head = paged ? a.page_head : own->to.head * int64_t(sizeof(T));
  char* const to = (paged ? const_cast<char*>(own->pages) + block * own->block
                          : own->to.base) +
                   (paged ? inside : token) * to_token + first_head * to_head;
  // distances inside a workgroup are mostly 32-bit
  const bool near = max(max(from_token, to_token) * count, max(from_head, to_head) * heads) <
                    (int64_t(1) << 30);
  const auto distance = [&](int32_t t, int64_t token_bytes, int32_t head, int64_t head_bytes) {
    return near ? int64_t(static_cast<uint32_t>(t) * static_cast<uint32_t>(token_bytes) +
                          static_cast<uint32_t>(head) * static_cast<uint32_t>(head_bytes))
                : t * token_bytes + head * head_bytes;
  };

  // A lane's items are kPlaceLanes apart; their places go along by sums. Of a head, N values
  // from `at` and N from `next`.
  struct Item {
    int32_t t, head, unit;
  };
  const int32_t step_rows = quotient(kPlaceLanes, a.units);
  const int32_t step_units = kPlaceLanes - step_rows * units;
  const int32_t step_t = step_rows / heads, step_heads = step_rows - step_t * heads;
  const auto advance = [&](Item& m) {
    m.unit += step_units;
    const bool row = m.unit >= units;
    m.unit -= row ? units : 0;
    m.head += step_heads + row;
    const bool wraps = m.head >= heads;
    m.head -= wraps ? heads : 0;
    m.t += step_t + wraps;
  };
  const int32_t turned_units = turned ? a.pairs / N : 0;
  const auto places = [&](const Item& m, int32_t* at, int32_t* next) {
    const bool turn = m.unit < turned_units;
    if (N == 1 && turn && a.interleaved) {
      *at = 2 * m.unit;
      *next = *at + 1;
    } else {
      *at = turn ? N * m.unit : rest + N * m.unit;
      *next = *at + (turn ? a.pairs : a.head_dim / 2 - rest);
    }
    return turn;
  };

  // Values stay as they came until they are needed: made wider at once, each item's loads
  // would be waited for before the next one's, and all before the angles.
  // Items on their way together: of 16-bit values, 16,000 tokens of 32 heads (three sets in
  // turn) take 50 us by two and 47 by three or four; of 32 bits, prompts take 213 by one to
  // three, 217 by four.
  constexpr int kItems = N == 8 ? 3 : 2;
  constexpr bool kAlike = sizeof(T) == sizeof(G);
  Raw<N, G> x[kItems], y[kItems];
  Raw<N, T> xq[kItems], yq[kItems];     // (queries, where they are of another size)
  const auto take = [&](int u, const Item& m) {
    int32_t at, next;
    places(m, &at, &next);
    const char* row = from + distance(m.t, from_token, m.head, from_head);
    if (kAlike || !query) {
      x[u].load(reinterpret_cast<const G*>(row) + at, words, lines);
      y[u].load(reinterpret_cast<const G*>(row) + next, words, lines);
    } else {
      xq[u].load(reinterpret_cast<const T*>(row) + at, words, lines);
      yq[u].load(reinterpret_cast<const T*>(row) + next, words, lines);
    }
  };
  int32_t i = threadIdx.x;
  Item item[kItems];
  item[0].unit = i - quotient(i, a.units) * units;
  item[0].t = quotient(i, a.units) / heads;
  item[0].head = quotient(i, a.units) - item[0].t * heads;
#pragma unroll
  for (int u = 1; u < kItems; ++u) {
    item[u] = item[u - 1];
    advance(item[u]);
  }
#pragma unroll
  for (int u = 0; u < kItems; ++u)
    if (i + u * kPlaceLanes < items) take(u, item[u]);

  if (turned) {
    for (int32_t j = threadIdx.x; j < count * a.pairs; j += kPlaceLanes) {
      const int32_t t = quotient(j, a.by_pairs), pair = j - t * a.pairs;
      int64_t p = position + t;
      if (a.positions)
        p = a.position_bytes == 8 ? static_cast<const int64_t*>(a.positions)[token + t]
                                  : static_cast<const int32_t*>(a.positions)[token + t];
      double turn = static_cast<double>(p) * a.turns[pair];
      turn -= rint(turn);
      float s, c;
      sincospif(static_cast<float>(2 * turn), &s, &c);
      cosine[j] = c * a.amplitude;
      sine[j] = s * a.amplitude;
    }
  }
  __syncthreads();
  for (; i < items; i += kItems * kPlaceLanes) {
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      if (i + u * kPlaceLanes >= items) continue;
      const Item& m = item[u];
      int32_t at, next;
      const bool turn = places(m, &at, &next);
      float p[N], r[N];
      if (query) {
        Raw<N, T> px, py;
        if constexpr (kAlike) {
          __builtin_memcpy(px.w, x[u].w, sizeof px.w);
          __builtin_memcpy(py.w, y[u].w, sizeof py.w);
        } else {
          px = xq[u];
          py = yq[u];
        }
        px.widen(p);
        py.widen(r);
      } else {
        x[u].widen(p);
        y[u].widen(r);
      }
      if (turn) {
        const float* c = cosine + m.t * a.pairs;
        const float* s = sine + m.t * a.pairs;
        if (!a.interleaved || N == 1) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            turn_pair(p[j], r[j], c[N * m.unit + j], s[N * m.unit + j]);
        } else if constexpr (N > 1) {
#pragma unroll
          for (int j = 0; j < N / 2; ++j) {
            const int pair = at / 2 + j, other = next / 2 + j;
            turn_pair(p[2 * j], p[2 * j + 1], c[pair], s[pair]);
            turn_pair(r[2 * j], r[2 * j + 1], c[other], s[other]);
          }
        }
      }
      // all that is written is of type T; without a plan, T is G
      T* const row = reinterpret_cast<T*>(to + distance(m.t, to_token, m.head, to_head));
      Raw<N, T> out;
      out.round(p);
      out.store(row + at, to_words, to_lines);
      out.round(r);
      out.store(row + next, to_words, to_lines);
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
#pragma unroll
      for (int s = 0; s < kItems; ++s) advance(item[u]);
      if (i + (kItems + u) * kPlaceLanes < items) take(u, item[u]);
    }
  }
}

// --------------------------------------------------------------- attention --

struct PagedAttendArgs {
  Sight sight;
  Pages pages;
  const char* plan;
  int64_t at_table, at_items, at_merges;
  Values q, out;
  float* lse;           // null: not asked for
  int64_t lse_token;
  float* work;          // parts of this kind's items, by slot
  int64_t slot_floats;
  int64_t kind_work[kKinds];   // merge: where each kind's parts begin
  float* work_base;
  int64_t kind_slot_floats[kKinds];
  int32_t group, kind;
};

typedef const AEGKV_CONSTANT PagedAttendArgs* PagedCold;
typedef const AEGKV_CONSTANT Item* PagedItem;

__device__ __forceinline__ PagedCold paged_cold() {
  return anew((PagedCold)__builtin_amdgcn_kernarg_segment_ptr());
}

// A row's running sum is taken against a score near its largest one, and only a
// probability past kLimit has the row looked through for its largest: 2^kLift
// stands for `top`. A product's score of thousands would be lost beside `lift`
// beyond kLimit; such rows, and those without a score yet, take each tile the long
// way, against their largest score itself. `sum` is the lane's own part, of the unrounded
// probabilities (log-sum-exps are made of it), 32 bits.
struct RowSum {
  float top = -INFINITY;
  float lift = 1e30f;    // kLift - top * c; past kLimit while there is no top
  float sum = 0.f;
};

// log2 of what sums are taken against: exactly what the exponents had added. A row
// without a score has nothing to compare: its base is below any that scores make.
template <typename T>
__device__ __forceinline__ float row_base(const RowSum& s, float c) {
  if (s.top == -INFINITY) return s.top;
  return fabsf(s.lift) > Matrix<T>::kLimit ? s.top * c - Matrix<T>::kLift : -s.lift;
}

// N scores of a row (x, -inf where hidden) into probabilities in place; `most_of` is the
// largest of a value over the lanes that share the row, O their output sums.
template <typename T, int N, typename M, typename O, int K>
__device__ __forceinline__ void softmax_part(float (&x)[N], float c, RowSum& s, O (&o)[K],
                                             const M& most_of) {
  float e[N];
  const auto exponents = [&](float from, float lift) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i] - from, c, lift));
  };
  const auto largest_of = [](const float (&y)[N]) {
    float m = y[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, y[i]);
    return m;
  };
  exponents(0.f, s.lift);
  if (__any(fmaxf(largest_of(e), fabsf(s.lift)) > Matrix<T>::kLimit)) {
    const float most = fmaxf(s.top, most_of(largest_of(x)));
    const float fade = s.top == most ? 1.f : __builtin_amdgcn_exp2f((s.top - most) * c);
    s.sum *= fade;
#pragma unroll
    for (int d = 0; d < K; ++d) o[d] *= fade;
    s.top = most;
    if (most != -INFINITY) s.lift = Matrix<T>::kLift - most * c;
    const bool far = (fabsf(s.lift) > Matrix<T>::kLimit) & (most != -INFINITY);
    exponents(far ? most : 0.f, far ? Matrix<T>::kLift : s.lift);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sum += e[i];
    x[i] = e[i];
  }
  s.sum += sum;
}

// Probabilities as the second product's operand. The matrix units take 16 bits, so each is
// rounded once (the row's sum, and with it the log-sum-exp, is of the unrounded ones): a
// result is off by at most half a step of the sum of probability times |V|, as much again as
// its own rounding. 64 decodes in bfloat16 are 0.0021 off, of the size of their results; with
// a second product over what the rounding leaves 0.0017, what rounding the exact results gives,
// but then 64 decodes take 222 us instead of 177, two long contexts 104 instead of 82, and
// four prompts 249 instead of 195.
template <typename T, int N>
__device__ __forceinline__ typename Matrix<T>::v8 round8(const float (&x)[N], int from) {
  typename Matrix<T>::v8 p;
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = static_cast<T>(x[from + i]);
  return p;
}

template <typename T, typename P>
__device__ __forceinline__ T* paged_result_row(PagedCold args, P it, int32_t row) {
  const int32_t group = args->group, token = row / group;
  return reinterpret_cast<T*>(args->out.base) + (int64_t(it->token) + token) * args->out.token +
         (int64_t(it->kv_head) * group + (row - token * group)) * args->out.head;
}

template <typename P>
__device__ __forceinline__ void store_lse(PagedCold args, P it, int32_t row, float base,
                                          float sum) {
  if (!args->lse) return;
  const int32_t group = args->group, token = row / group;
  args->lse[(int64_t(it->token) + token) * args->lse_token + int64_t(it->kv_head) * group +
            (row - token * group)] = 0.6931471805599453f * (base + __builtin_amdgcn_logf(sum));
}

// A query row's eight values from `at` on.
template <typename T>
__device__ __forceinline__ v4u query8(PagedCold args, PagedItem it, int32_t row, bool there,
                                      int32_t at) {
  v4u x = {0, 0, 0, 0};
  if (there) {
    const int32_t group = args->group, token = row / group;
    const T* from = reinterpret_cast<const T*>(args->q.base) +
                    (int64_t(it->token) + token) * args->q.token +
                    (int64_t(it->kv_head) * group + (row - token * group)) * args->q.head + at;
    if (args->q.whole_words) {
      x = *(const gv4u*)from;
    } else {
      T t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = from[j];
      __builtin_memcpy(&x, t, 16);
    }
  }
  return x;
}

// Bits 15 and 31 of the result: whether a word's lower and upper value are infinities
// or no numbers (an exponent of ones carries into the sign's place).
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr bool kWide = std::is_same<T, __bf16>::value;
  return (w & (kWide ? 0x7F807F80u : 0x7C007C00u)) + (kWide ? 0x00800080u : 0x04000400u);
}
constexpr uint32_t kNotFinite = 0x80008000u;

// All bits of the values that not_finite() found.
__device__ __forceinline__ uint32_t whole_values(uint32_t found) {
  return ((found >> 15) & 0x00010001u) * 0xFFFFu;
}

// Where a half tile of 16 tokens lies for one head: the same for the whole wave.
struct PagedHalf {
  const char* k;
  const char* v;
};

__device__ __forceinline__ PagedHalf paged_half(const Pages& p, int32_t kv_head, int block_shift,
                                                int32_t block, int32_t position) {
  const int64_t inside = int64_t(position & ((1 << block_shift) - 1)) * p.token +
                         int64_t(kv_head) * p.head;
  return PagedHalf{p.k + block * p.k_block + inside, p.v + block * p.v_block + inside};
}

constexpr int kPagedLanes = 256, kPagedWaves = 4;

// Waves a SIMD has to hold, as the registers allow.
template <int D, int R>
constexpr int kPagedPerSimd = D <= 128 && R == 1 ? 3 : D <= 128 ? 2 : 1;

template <int D, int R>
struct PagedJoin {
  float part[kPagedWaves][16][D + 4];
  float base[kPagedWaves][16 * R], sum[kPagedWaves][16 * R];
};

// A lane's part of a tile of 32 tokens (m = l % 16, g = l / 16). Of K, for both
// halves of 16 tokens, token m's values 32 s + 8 g .. + 7 of each matrix step s. Of V
// the values [D/16 m, D/16 (m + 1)) of tokens 4 g .. 4 g + 3 of each half: the
// tokens that the lane's probabilities belong to, so that these are the second
// product's operand as they are; eight tokens of a value come side by side by
// byte permutes. K comes through the caches, 64 bytes of a row at a time (two contexts
// of 100,000 tokens, 4 KV heads of 28: 73 us, past them 80), V, whole rows, past them.
template <int D>
struct PagedTile {
  static constexpr int kRun = D / 16, kWords = kRun / 2;
  v4u k[2][D / 32];
  uint32_t v[2][4][kWords];

  __device__ __forceinline__ void load_k(const PagedHalf* h, int32_t token, uint32_t m,
                                         uint32_t g) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
        load_bytes<16, false>(reinterpret_cast<uint32_t*>(&k[i][s]), h[i].k,
                             m * token + g * 16 + s * 64);
  }
  __device__ __forceinline__ void load_v(const PagedHalf* h, int32_t token, uint32_t m,
                                         uint32_t g) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (uint32_t t = 0; t < 4; ++t)
        load_bytes<kRun * 2, true>(v[i][t], h[i].v, (4 * g + t) * token + m * (kRun * 2));
  }

  // In a tile that some row does not see whole: what no row of [low, high] sees may
  // hold anything, and its product with a probability of 0 has to be 0. Returns the
  // seen tokens (bit 4 half + t) with infinities or no numbers among the lane's values;
  // they count as 0 too, and add_odd adds them for the rows that see them.
  template <typename T>
  __device__ __forceinline__ uint32_t clear(int32_t begin, int32_t g, int32_t low, int32_t high,
                                            const Sight& a) {
    uint32_t odd = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t found = 0;
#pragma unroll
        for (int w = 0; w < kWords; ++w) found |= not_finite<T>(v[half][t][w]);
        const bool bad = (found & kNotFinite) != 0;
        const int32_t j = begin + 16 * half + 4 * g + t;
        const bool any = (j <= high) & ((low - j < a.window) | (j < a.sinks));
        odd |= (bad & any) ? 1u << (4 * half + t) : 0u;
        const uint32_t keep = bad ? 0u : ~0u;
#pragma unroll
        for (int w = 0; w < kWords; ++w) v[half][t][w] &= keep;
      }
    return odd;
  }

  // The operands of values 2 B and 2 B + 1: eight tokens side by side each.
  template <typename T, int B>
  __device__ __forceinline__ void operands(typename Matrix<T>::v8* even,
                                           typename Matrix<T>::v8* odd) const {
    uint32_t e[4], o[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t c0 = v[t / 2][2 * (t % 2)][B], c1 = v[t / 2][2 * (t % 2) + 1][B];
      e[t] = __builtin_amdgcn_perm(c1, c0, 0x05040100u);
      o[t] = __builtin_amdgcn_perm(c1, c0, 0x07060302u);
    }
    __builtin_memcpy(even, e, 16);
    __builtin_memcpy(odd, o, 16);
  }
};

// Adds, in 32 bits and to the rows that see them, the values that clear() took out of a
// tile (they are rare): lanes_of(odd, t) are the runs of token t that were cleared.
template <int D, typename T, int R>
__device__ __forceinline__ void add_odd(const Sight& a, const Pages& pages, uint32_t odd,
                                        const AEGKV_CONSTANT int32_t* table, int32_t kv_head,
                                        int32_t begin, const int32_t* position, int m, int g,
                                        const typename Matrix<T>::v8* p, f32x4 (*o)[D / 16]) {
  constexpr int kRun = D / 16;
#pragma unroll 1
  for (int t = 0; t < kTile; ++t) {
    const uint32_t lanes = lanes_of(odd, t);
    if (!lanes) continue;
    // nothing of this is held in registers while there are no such tokens
    int first = 4 * g, row = m;
    asm volatile("" : "+v"(first), "+v"(row));
    const int32_t j = begin + t;
    const PagedHalf h = paged_half(pages, kv_head, a.block_shift, table[j >> a.block_shift], j);
    float weight[R];
    bool sees[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint32_t w[4];
      __builtin_memcpy(w, &p[r], 16);
      const int word = 2 * (t / 16) + t % 4 / 2;
      const uint32_t pair = static_cast<uint32_t>(
          __shfl(static_cast<int>(word < 2 ? (word ? w[1] : w[0]) : (word == 2 ? w[2] : w[3])),
                 16 * (t % 16 / 4) + row));
      weight[r] = static_cast<float>(
          __builtin_bit_cast(T, static_cast<uint16_t>(t % 2 ? pair >> 16 : pair)));
      sees[r] = seen(a, position[r], j);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int run = first + i;
      const bool here = (lanes >> run) & 1;
      const T* v = reinterpret_cast<const T*>(h.v) + run * kRun;
#pragma unroll
      for (int d = 0; d < kRun; ++d) {
        const float x = static_cast<float>(v[d]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float was = o[r][d][i];
          o[r][d][i] = (here & sees[r]) ? __builtin_fmaf(weight[r], x, was) : was;
        }
      }
    }
  }
}

// Single tokens and short runs: S^T = K Q^T and O^T = V^T P^T over tiles of 32
// tokens, one pass; the four waves take the item's tiles in turn and join at its end.
// A row's state is its lane's, its probabilities the second product's operand as they lie.
// Bound by HBM: 64 requests of 8 KV heads (1.04 GB) take 172 us and their parts 5 to
// join, 5.9 TB/s in all; with eight spilled registers it took 201.
template <int D, typename T, int R>
__device__ __forceinline__ void paged_attend_item(const Sight& a, const Pages& pages,
                                                  PagedItem it, PagedJoin<D, R>& share) {
  typedef typename Matrix<T>::v8 v8;
  constexpr int kSteps = D / 32, kOut = D / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, m = lane % 16, g = lane / 16;
  const PagedCold args = paged_cold();
  const auto* table = in_plan<int32_t>(args->plan, args->at_table) + it->table;
  const Tiles tiles = {it->first_tiles, it->window_tile - it->first_tiles, it->tile_end};
  const int32_t kv_head = it->kv_head;

  struct Blocks {
    int32_t position, block[2];
  };
  const auto find = [&](int32_t v) {
    Blocks b;
    b.position = tiles.at(min(v, tiles.end - 1)) * kTile;
    b.block[0] = table[b.position >> a.block_shift];
    b.block[1] = table[(b.position + 16) >> a.block_shift];
    return b;
  };
  PagedHalf h[2];
  const auto halves = [&](const Blocks& b) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      h[i] = paged_half(pages, kv_head, a.block_shift, b.block[i], b.position + 16 * i);
  };
  PagedTile<D> t;
  int32_t at = it->tile + wave;
  if (at < tiles.end) {
    halves(find(at));
    t.load_k(h, pages.token, m, g);
    t.load_v(h, pages.token, m, g);
  }
  Blocks ahead = find(at + kPagedWaves);

  v8 q[R][kSteps];
  int32_t position[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool there = 16 * r + m < it->rows;
    position[r] = it->base + (there ? (it->row + 16 * r + m) / args->group : 0);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const v4u x = query8<T>(args, it, it->row + 16 * r + m, there, 32 * s + 8 * g);
      __builtin_memcpy(&q[r][s], &x, 16);
    }
  }
  const int32_t low = it->base + it->row / args->group;
  const int32_t high = it->base + (it->row + it->rows - 1) / args->group;

  f32x4 o[R][kOut];
  RowSum state[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int d = 0; d < kOut; ++d) o[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (; at < tiles.end; at += kPagedWaves) {
    const int32_t begin = tiles.at(at) * kTile;
    const bool more = at + kPagedWaves < tiles.end;
    // scores: lane holds row m, tokens 4g + i of both halves
    f32x4 x[R][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        v8 k;
        __builtin_memcpy(&k, &t.k[half][s], 16);
#pragma unroll
        for (int r = 0; r < R; ++r) x[r][half] = Matrix<T>::mma(k, q[r][s], x[r][half]);
      }
    }
    if (more) {
      halves(ahead);
      t.load_k(h, pages.token, m, g);
    }
    ahead = find(at + 2 * kPagedWaves);

    uint32_t odd = 0;
    float e[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) e[r][i] = x[r][i / 4][i % 4];
    if (!seen_whole(a, low, high, begin)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r)
          e[r][i] = seen(a, position[r], begin + 16 * (i / 4) + 4 * g + i % 4) ? e[r][i]
                                                                               : -INFINITY;
      odd = t.template clear<T>(begin, g, low, high, a);
    }
    v8 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      softmax_part<T>(e[r], a.c, state[r], o[r], [](float v) { return row_max(v); });
      p[r] = round8<T>(e[r], 0);
    }
    each_constant<0, kOut / 2>([&](auto b) {
      constexpr int B = decltype(b)::value;
      v8 first, second;
      t.template operands<T, B>(&first, &second);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        o[r][2 * B] = Matrix<T>::mma(first, p[r], o[r][2 * B]);
        o[r][2 * B + 1] = Matrix<T>::mma(second, p[r], o[r][2 * B + 1]);
      }
    });
    if (__any(odd != 0))
      add_odd<D, T, R>(a, pages, odd, table, kv_head, begin, position, m, g, p, o);
    if (more) t.load_v(h, pages.token, m, g);
  }

  // join the waves: each scales its part to the largest of their bases
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float s = state[r].sum;
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (g == 0) {
      share.base[wave][16 * r + m] = row_base<T>(state[r], a.c);
      share.sum[wave][16 * r + m] = s;
    }
  }
  __syncthreads();
  const PagedCold end_args = paged_cold();
  const PagedItem ended = anew(it);
  constexpr int kRowLanes = 16, kEach = D / kRowLanes;   // of a row, values of each
  const int row = threadIdx.x / kRowLanes, part = threadIdx.x % kRowLanes;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float most = share.base[0][16 * r + m];
#pragma unroll
    for (int w = 1; w < kPagedWaves; ++w) most = fmaxf(most, share.base[w][16 * r + m]);
    const float base = share.base[wave][16 * r + m];
    const float fade = base == most ? 1.f : __builtin_amdgcn_exp2f(base - most);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kOut; ++d)
        share.part[wave][m][(D / 16) * (4 * g + i) + d] = o[r][d][i] * fade;
    __syncthreads();
    float y[kEach] = {};
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) y[i] += share.part[w][row][part * kEach + i];
    }
    if (r + 1 < R) __syncthreads();   // before the next row tile's parts
    if (16 * r + row < ended->rows) {
      float all = share.base[0][16 * r + row], total = 0.f;
#pragma unroll
      for (int w = 1; w < kPagedWaves; ++w) all = fmaxf(all, share.base[w][16 * r + row]);
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w) {
        const float b = share.base[w][16 * r + row];
        total += share.sum[w][16 * r + row] *
                 (b == all ? 1.f : __builtin_amdgcn_exp2f(b - all));
      }
      if (ended->slot < 0) {
        T* to = paged_result_row<T>(end_args, ended, ended->row + 16 * r + row);
        const float inv = 1.f / total;
#pragma unroll
        for (int i = 0; i < kEach; ++i) to[part * kEach + i] = static_cast<T>(y[i] * inv);
        if (part == 0) store_lse(end_args, ended, ended->row + 16 * r + row, all, total);
      } else {
        float* to = end_args->work + ended->slot * end_args->slot_floats + (16 * r + row) * (D + 4);
#pragma unroll
        for (int i = 0; i < kEach; ++i) to[part * kEach + i] = y[i];
        if (part == 0) {
          to[D] = all;
          to[D + 1] = total;
        }
      }
    }
  }
}

template <int D, typename T, int R>
__global__ __launch_bounds__(kPagedLanes, (kPagedPerSimd<D, R>)) void paged_attend_kernel(
    PagedAttendArgs args) {
  __shared__ PagedJoin<D, R> joined;
  const Sight sight = args.sight;
  const Pages pages = args.pages;
  const PagedItem it = in_plan<Item>(args.plan, args.at_items) + blockIdx.x;
  if (static_cast<int32_t>(blockIdx.x) >= in_plan<Header>(args.plan, 0)->items[args.kind]) return;
  paged_attend_item<D, T, R>(sight, pages, it, joined);
}

// largest of a value over the two lanes of a row (l, l ^ 32)
__device__ __forceinline__ float pair_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// Prompts: 128 rows a workgroup, 32 a wave, as the above with products of 32 x 32.
// Tiles of 32 tokens go straight from the cache to a ring of four in shared memory, as
// rows of 16-byte chunks, each row's chunks exchanged by its number so that neither
// product's reads meet in a bank: K's operands are a token's chunk a lane, V's come four
// tokens of a value a lane by transposing reads. Lane l (row l % 32, h = l / 32) holds the
// scores of tokens 8 (i / 4) + 4 h + i % 4, i < 16, and they are the second product's
// operand as they lie. Three tiles are in work at once: the second product of one beside
// the scores of the next and the exponents between them. Bound by what two waves a SIMD
// issue: matrix units are busy 48 % of a long prompt's time, the vector unit 50. Four
// prompts of 1,000 to 4,096 tokens, 8 KV heads of 32, take 195 to 205 us 128 wide (770 to 810
// TFLOP/s), 121 64 wide (650) and 430 256 wide (735, one wave a SIMD: a CU holds one ring),
// and one of 32,768 runs at 1,055, 890 and 965. With registers instead of the ring the four
// took 208, a tile after another without its order of issue 193, where this took 188.
constexpr int kRing = 4, kRowsWave = 32, kTileRowsWave = kTile / kPagedWaves;
static_assert(kManyRows == kPagedWaves * kRowsWave, "rows of a workgroup");

template <int D>
struct PagedRing {
  static constexpr int kChunks = D / 8;    // of 16 bytes in a row
  v4u k[kRing][kTile * kChunks];
  v4u v[kRing][kTile * kChunks];
  static __device__ __forceinline__ int k_turn(int token) {
    return D == 64 ? token / 2 % 8 : token % 16;
  }
  static __device__ __forceinline__ int v_turn(int token) { return 2 * (token % 4); }
  static __device__ __forceinline__ int k_at(int token, int chunk) {
    return token * kChunks + (chunk ^ k_turn(token));
  }
  static __device__ __forceinline__ int v_at(int token, int chunk) {
    return token * kChunks + (chunk ^ v_turn(token));
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Of 16 lanes that point at four rows of 16 values, four values a lane: lane i gets
// value i of the four rows.
__device__ __forceinline__ s16x4 read_turned(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)static_cast<uintptr_t>(at));
}

__device__ __forceinline__ uint32_t shared_address(const v4u* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const v4u*)p));
}

// 16 bytes a lane from `base` (the same for the wave) + offset to shared memory, lane
// after lane from `to` on, which the instruction takes from m0; NT: past the caches. The
// compiler does not know that shared memory changes: whoever reads it waits for the loads
// first. (Told of it, it waits for all such loads before any read of shared memory.)
template <bool NT = false>
__device__ __forceinline__ void load_shared(const char* base, uint32_t offset, const v4u* to) {
  if constexpr (NT)
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :: "v"(offset), "s"(base), "{m0}"(shared_address(to)) : "memory");
  else
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(offset), "s"(base), "{m0}"(shared_address(to)) : "memory");
}

// All of the wave's loads have come but the last LATER, its reads of shared memory too,
// and the other waves are here as well.
template <int LATER>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(LATER) : "memory");
}

// Adds, in 32 bits and to the rows that see their tokens, the infinities and no numbers
// that were taken out of a tile's V (they are rare).
template <int D, typename T>
__device__ __forceinline__ void add_odd_rows(const Sight& a, const v4u* tile, int32_t begin,
                                             int32_t low, int32_t high, int32_t position, int n,
                                             int h, const float (&e)[16], f32x16 (&o)[D / 32]) {
#pragma unroll 1
  for (int t = 0; t < kTile; ++t) {
    const int32_t j = begin + t;
    if (!((j <= high) & ((low - j < a.window) | (j < a.sinks)))) continue;   // none sees it
    const bool sees = seen(a, position, j);
    // the row's probability of token t, from the lane that has it
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      mine = i == 4 * (t / 8) + t % 4 ? static_cast<float>(static_cast<T>(e[i])) : mine;
    const float weight = __shfl(mine, n + 32 * (t / 4 % 2));
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int value = 32 * d + 8 * (i / 4) + 4 * h + i % 4;
        const T y = reinterpret_cast<const T*>(
            &tile[PagedRing<D>::v_at(t, value / 8)])[value % 8];
        const bool bad = not_finite<T>(__builtin_bit_cast(uint16_t, y)) & kNotFinite;
        const float was = o[d][i];
        o[d][i] = (bad & sees) ? __builtin_fmaf(weight, static_cast<float>(y), was) : was;
      }
  }
}

template <int D, typename T>
__device__ __forceinline__ void paged_prompt_item(const Sight& a, const Pages& pages,
                                                  PagedItem it, PagedRing<D>& ring) {
  typedef typename Matrix<T>::v8 v8;
  typedef PagedRing<D> Ring;
  constexpr int kSteps = D / 16, kOut = D / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, n = lane % 32, h = lane / 32;
  const PagedCold args = paged_cold();
  const auto* table = in_plan<int32_t>(args->plan, args->at_table) + it->table;
  const Tiles tiles = {it->first_tiles, it->window_tile - it->first_tiles, it->tile_end};
  const int32_t group = args->group, kv_head = it->kv_head;
  const int32_t first = it->tile, end = it->tile_end;

  // This wave's share of a tile: eight tokens of K and of V. Lane by lane the places of
  // shared memory are given; which chunk of the row comes there follows from them.
  constexpr int kLoads = kTileRowsWave * Ring::kChunks / 64;
  uint32_t k_from[kLoads], v_from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int slot = i * 64 + lane, row = slot / Ring::kChunks, at = slot % Ring::kChunks;
    const int token = wave * kTileRowsWave + row;
    k_from[i] = token % 16 * pages.token + (at ^ Ring::k_turn(token)) * 16;
    v_from[i] = token % 16 * pages.token + (at ^ Ring::v_turn(token)) * 16;
  }
  // The block of the tile that is fetched next is looked up a tile before.
  struct Where {
    int32_t position, block;
  };
  const auto look_up = [&](int32_t t) {
    // behind the last tile the last one comes again, and is not used
    const int32_t at = tiles.at(min(t, end - 1)) * kTile + 16 * (wave / 2);
    return Where{at, table[at >> a.block_shift]};
  };
  const auto fetch = [&](int32_t t, const Where& from) {
    const PagedHalf half = paged_half(pages, kv_head, a.block_shift, from.block, from.position);
    const int slot = (t - first) & (kRing - 1), at = wave * kTileRowsWave * Ring::kChunks;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_shared(half.k, k_from[i], &ring.k[slot][at + i * 64]);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_shared(half.v, v_from[i], &ring.v[slot][at + i * 64]);
  };
  const Where begin[3] = {look_up(first), look_up(first + 1), look_up(first + 2)};
  Where ahead = look_up(first + 3);

  const int32_t row0 = it->row + wave * kRowsWave;
  const int32_t rows = min(max(it->rows - wave * kRowsWave, 0), kRowsWave);
  const int32_t low = it->base + row0 / group;
  const int32_t high = rows ? it->base + (row0 + rows - 1) / group : -1;
  const bool there = n < rows;
  const int32_t position = there ? it->base + (row0 + n) / group : low;
  v8 q[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const v4u x = query8<T>(args, it, row0 + n, there, 16 * s + 8 * h);
    __builtin_memcpy(&q[s], &x, 16);
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) fetch(first + i, begin[i]);

  f32x16 o[kOut];
#pragma unroll
  for (int d = 0; d < kOut; ++d) o[d] = f32x16{};
  RowSum state;

  // Three tiles are in work at once, so that the matrix unit has products while
  // exponentials are made: the scores of tile t + 1, the softmax of t, the output of t - 1.
  v8 k[kSteps], p[2];
  uint32_t v[2][kOut][4];
  const auto read_k = [&](int32_t t) {
    const v4u* from = ring.k[(t - first) & (kRing - 1)];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      __builtin_memcpy(&k[s], &from[Ring::k_at(n, 2 * s + h)], 16);
  };
  // Where a lane reads V turned: token (lane % 16) / 4 of four, 4 values of 16, in the row's
  // chunks of an even and of an odd run of 32 values; all else is added by number. V's
  // operand: tokens 16 ks + 4 h + j and 16 ks + 8 + 4 h + j of a value.
  uint32_t v_place[2];
#pragma unroll
  for (int d = 0; d < 2; ++d)
    v_place[d] = shared_address(ring.v[0]) + 8 * (lane % 2) +
                 16 * Ring::v_at(4 * h + lane % 16 / 4,
                                 4 * d + 2 * (lane / 16 % 2) + lane % 4 / 2);
  const auto read_v = [&](int32_t t) {
    const uint32_t slot = ((t - first) & (kRing - 1)) * sizeof ring.v[0];
    const uint32_t place[2] = {v_place[0] + slot, v_place[1] + slot};
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int d = 0; d < kOut; ++d)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const s16x4 y = read_turned(place[d % 2] + 16 * ((16 * ks + 8 * j) * Ring::kChunks +
                                                           8 * (d / 2)));
          __builtin_memcpy(&v[ks][d][2 * j], &y, 8);
        }
  };
  const auto scores = [&]() {
    f32x16 x = {};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) x = Matrix<T>::mma32(k[s], q[s], x);
    return x;
  };
  const auto outputs = [&]() {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int d = 0; d < kOut; ++d) {
        v8 y;
        __builtin_memcpy(&y, v[ks][d], 16);
        o[d] = Matrix<T>::mma32(y, p[ks], o[d]);
      }
  };
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    p[ks] = v8{};
#pragma unroll
    for (int d = 0; d < kOut; ++d)
#pragma unroll
      for (int w = 0; w < 4; ++w) v[ks][d][w] = 0;
  }

  wait_and_meet<2 * 2 * kLoads>();
  read_k(first);
  f32x16 x = scores();
  for (int32_t t = first; t < end; ++t) {
    wait_and_meet<2 * kLoads>();
    read_k(t + 1);
    fetch(t + 3, ahead);
    ahead = look_up(t + 4);
    const int32_t begin = tiles.at(t) * kTile;
    const bool whole = seen_whole(a, low, high, begin);
    float e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = x[i];
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        e[i] = seen(a, position, begin + 8 * (i / 4) + 4 * h + i % 4) ? e[i] : -INFINITY;
    }
    outputs();
    x = scores();
    read_v(t);
    // a product, two instructions and an exponential in turn
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
    }
    softmax_part<T>(e, a.c, state, o, [](float y) { return pair_max(y); });
    if (!whole) {
      // infinities and no numbers: a probability of 0 would make no number of them
      uint32_t found = 0;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) found |= not_finite<T>(v[ks][d][w]);
      if (__any((found & kNotFinite) != 0)) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int d = 0; d < kOut; ++d)
#pragma unroll
            for (int w = 0; w < 4; ++w)
              v[ks][d][w] &= ~whole_values(not_finite<T>(v[ks][d][w]));
        add_odd_rows<D, T>(a, ring.v[(t - first) & (kRing - 1)], begin, low, high, position, n,
                           h, e, o);
      }
    }
    p[0] = round8<T>(e, 0);
    p[1] = round8<T>(e, 8);
  }
  outputs();

  const PagedCold end_args = paged_cold();
  const PagedItem ended = anew(it);
  const int32_t slot = ended->slot;
  const float total = state.sum + __shfl_xor(state.sum, 32);
  if (!there) return;
  const float base = row_base<T>(state, a.c);
  float* part = end_args->work + slot * end_args->slot_floats +
                (row0 + n - ended->row) * (D + 4);
  T* to = paged_result_row<T>(end_args, ended, row0 + n);
  const float inv = slot < 0 ? 1.f / total : 1.f;
#pragma unroll
  for (int d = 0; d < kOut; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int value = 32 * d + 8 * i + 4 * h;
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = o[d][4 * i + j] * inv;
      if (slot >= 0) {
        __builtin_memcpy(part + value, y, 16);
      } else {
        T r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = static_cast<T>(y[j]);
        if (end_args->out.whole_words) {
          __builtin_memcpy(__builtin_assume_aligned(to + value, 8), r, 8);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) to[value + j] = r[j];
        }
      }
    }
  if (h == 0) {
    if (slot >= 0) {
      part[D] = base;
      part[D + 1] = total;
    } else {
      store_lse(end_args, ended, row0 + n, base, total);
    }
  }
}

template <int D, typename T>
__global__ __launch_bounds__(kPagedLanes, D == 256 ? 1 : 2) void paged_prompt_kernel(
    PagedAttendArgs args) {
  __shared__ PagedRing<D> ring;
  const Sight sight = args.sight;
  const Pages pages = args.pages;
  const PagedItem it = in_plan<Item>(args.plan, args.at_items) + blockIdx.x;
  if (static_cast<int32_t>(blockIdx.x) >= in_plan<Header>(args.plan, 0)->items[args.kind]) return;
  paged_prompt_item<D, T>(sight, pages, it, ring);
}

// Rows whose tiles several items shared: their parts, scaled to the largest base of
// all, over the sum of their sums. A workgroup's lanes are groups of D / 4,
// four values a lane. Of up to kMergeRows parts each group takes rows of its own;
// more (few rows over a long axis) are shared out to the groups, one row a workgroup.
// 4 to 6 us, of which 3 are a launch and the reads that follow one another.
template <int D, typename T>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttendArgs a) {
  constexpr int kLanes = D / 4, kSides = 256 / kLanes;
  __shared__ f32x4 side[kSides][kLanes];
  __shared__ float side_sum[kSides], side_top[4];
  const auto* mg = in_plan<Merge>(a.plan, a.at_merges) + blockIdx.x;
  if (static_cast<int32_t>(blockIdx.x) >= in_plan<Header>(a.plan, 0)->merges) return;
  const int64_t each = a.kind_slot_floats[mg->kind];
  const int32_t parts = mg->parts;
  const float* rows = a.work_base + a.kind_work[mg->kind] + mg->slot * each +
                      mg->first * (D + 4);
  const int at = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const auto store = [&](int32_t row, f32x4 y, float most, float total) {
    const PagedCold args = (PagedCold)__builtin_amdgcn_kernarg_segment_ptr();
    T* to = paged_result_row<T>(args, mg, mg->row + row) + 4 * at;
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = static_cast<T>(y[i] / total);
    if (at == 0) store_lse(args, mg, mg->row + row, most, total);
  };
  if (parts <= kMergeRows) {
    for (int32_t row = group; row < mg->rows; row += kSides) {
      const float* from = rows + row * (D + 4);
      float t[kMergeRows], most = -INFINITY;
#pragma unroll
      for (int p = 0; p < kMergeRows; ++p) {
        t[p] = p < parts ? from[p * each + D] : -INFINITY;
        most = fmaxf(most, t[p]);
      }
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
      float total = 0.f;
#pragma unroll
      for (int p = 0; p < kMergeRows; ++p) {
        if (p >= parts) continue;
        const float fade = t[p] == most ? 1.f : __builtin_amdgcn_exp2f(t[p] - most);
        y += *reinterpret_cast<const f32x4*>(from + p * each + 4 * at) * fade;
        total += from[p * each + D + 1] * fade;
      }
      store(row, y, most, total);
    }
    return;
  }
  float most = -INFINITY;
  for (int p = threadIdx.x; p < parts; p += 256) most = fmaxf(most, rows[p * each + D]);
#pragma unroll
  for (int far = 32; far; far /= 2) most = fmaxf(most, __shfl_xor(most, far));
  if (threadIdx.x % 64 == 0) side_top[threadIdx.x / 64] = most;
  __syncthreads();
  most = fmaxf(fmaxf(side_top[0], side_top[1]), fmaxf(side_top[2], side_top[3]));
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  float total = 0.f;
#pragma unroll 4
  for (int p = group; p < parts; p += kSides) {
    const float t = rows[p * each + D];
    const float fade = t == most ? 1.f : __builtin_amdgcn_exp2f(t - most);
    y += *reinterpret_cast<const f32x4*>(rows + p * each + 4 * at) * fade;
    total += rows[p * each + D + 1] * fade;
  }
  side[group][at] = y;
  if (at == 0) side_sum[group] = total;
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int i = 1; i < kSides; ++i) {
    y += side[i][at];
    total += side_sum[i];
  }
  store(0, y, most, total);
}

// --------------------------------------------------- weights of attention --

struct WeighArgs {
  Sight sight;
  Pages pages;
  const char* plan;
  int64_t at_seqs, at_table, at_place_tiles;
  Values q;
  const float* lse;
  int64_t lse_token;
  float* weights;       // [block][kv_head][token]
  Divisor group;
  int32_t kv_heads, first_tile;
};

constexpr int kWeighPlaces = kPlaceTile;

// One workgroup's work: places of one sequence under one KV head, and its queries.
struct WeighItem {
  int32_t kv_head, first;               // of the places
  int32_t len, base, rows, token, table;
  // Whether some query sees a place of [from, from + count).
  __device__ __forceinline__ bool reaches(const Sight& a, int32_t from, int32_t count) const {
    return (from < len) & ((base - (from + count - 1) < a.window) | (from < a.sinks));
  }
};

// MANY: of the sequences of more than kMostMore rows, whose tiles come first. A captured
// call has a workgroup for each tile that there is room for, and may find, after an
// update, a batch whose queries see one block in two places.
template <bool MANY>
__device__ __forceinline__ bool find_places(const WeighArgs& a, int32_t index, WeighItem* it) {
  const int32_t i = index / a.kv_heads, at = i + a.first_tile;
  const auto* h = in_plan<Header>(a.plan, 0);
  if (h->shared || at >= (MANY ? h->many_tiles : h->place_tiles) ||
      (!MANY && at < h->many_tiles))
    return false;
  const auto* tile = in_plan<PlaceTile>(a.plan, a.at_place_tiles) + at;
  const auto* s = in_plan<Seq>(a.plan, a.at_seqs) + tile->seq;
  it->kv_head = index - i * a.kv_heads;
  it->first = tile->first;
  it->len = s->len;
  it->base = s->len - s->fresh;
  it->rows = s->fresh * static_cast<int32_t>(a.group.by);
  it->token = s->token;
  it->table = s->table;
  return true;
}

// A query row's place among the values, and its log-sum-exp's.
__device__ __forceinline__ int64_t weigh_row(const WeighArgs& a, const WeighItem& it, int32_t row,
                                             int64_t token_stride, int64_t head_stride) {
  const int32_t token = quotient(row, a.group);
  return (int64_t(it.token) + token) * token_stride +
         (int64_t(it.kv_head) * a.group.by + (row - token * static_cast<int32_t>(a.group.by))) *
             head_stride;
}

// Eight values of a query row from `at` on. (Behind the last row, its own again: what comes
// of them is dropped.)
template <typename T>
__device__ __forceinline__ v4u weigh_query8(const WeighArgs& a, const WeighItem& it, int32_t row,
                                            int32_t at) {
  const T* from = reinterpret_cast<const T*>(a.q.base) +
                  weigh_row(a, it, min(row, it.rows - 1), a.q.token, a.q.head) + at;
  v4u x;
  __builtin_memcpy(&x, from, 16);
  return x;
}

// log2(e) times a row's log-sum-exp; infinity where there is no row: its share is 0.
__device__ __forceinline__ float row_log(const WeighArgs& a, const WeighItem& it, int32_t row) {
  const float x = a.lse[weigh_row(a, it, min(row, it.rows - 1), a.lse_token, 1)];
  return row < it.rows ? 1.4426950408889634f * x : INFINITY;
}

// A lane's place and what it has gathered before; asked for before its scores are made.
struct OwnPlace {
  float* to;
  float before;
  bool seen;
  // (a place behind the sequence's last one is the last one)
  __device__ __forceinline__ OwnPlace(const WeighArgs& a, const WeighItem& it, int32_t place,
                                      int64_t block) {
    const int32_t shift = a.sight.block_shift;
    seen = it.reaches(a.sight, place, 1);
    place = min(place, it.len - 1);
    to = a.weights + (((block * a.kv_heads + it.kv_head) << shift) +
                      (place & ((1 << shift) - 1)));
    before = place < it.base ? *to : 0.f;
  }
  __device__ __forceinline__ void add(float w) const {
    if (seen) *to = before + w;
  }
};

// w[place] += sum over the rows that see it of exp2(c s - log2(e) lse). A place
// belongs to one lane at the end: no atomics, and the sum's order is fixed. Up
// to 64 rows of a sequence: S = Q K^T by 16 x 16 x 32. Bound by HBM; what takes part is
// asked for at once, without branches. K comes straight to shared memory of the wave's own,
// whole rows at a time, and past the caches: into registers, a token a lane, each load
// takes half of a line, and most waves stand at a load that is not taken yet. 64 decodes of
// 100 to 8,000 tokens, 8 KV heads of 128, take 99 us (5.4 TB/s): 116 from registers, 110
// through the caches. A wave holds 8 KiB of K: with 64 places 105, with 16 100.
constexpr int weigh_parts(int head_dim) { return head_dim == 64 ? 4 : head_dim == 128 ? 2 : 1; }

template <int D, typename T>
__global__ __launch_bounds__(kPagedLanes, 4) void paged_weigh_kernel(WeighArgs a) {
  typedef typename Matrix<T>::v8 v8;
  constexpr int kSteps = D / 32, kParts = weigh_parts(D), kWavePlaces = 16 * kParts;
  constexpr int kShare = kWeighPlaces / (kPagedWaves * kWavePlaces);
  constexpr int kChunks = D / 8, kLoads = 16 * kChunks / 64;
  typedef PagedRing<D> Ring;
  __shared__ v4u held[kPagedWaves][kWavePlaces * kChunks];
  WeighItem it;
  const int32_t tile = blockIdx.x / (kShare * a.kv_heads);
  const int32_t rest = blockIdx.x - tile * kShare * a.kv_heads, share = rest / a.kv_heads;
  if (!find_places<false>(a, tile * a.kv_heads + rest - share * a.kv_heads, &it)) return;
  it.first += share * kPagedWaves * kWavePlaces;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, m = lane % 16, g = lane / 16;
  const int32_t begin = it.first + wave * kWavePlaces;
  if (!it.reaches(a.sight, begin, kWavePlaces)) return;
  const auto* table = in_plan<int32_t>(a.plan, a.at_table) + it.table;
  const int32_t last = it.len - 1, shift = a.sight.block_shift;
  // (parts behind the sequence's last place read its last one again)
  int32_t own_block = 0;
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    const int32_t at = min(begin + 16 * p, last & ~15);
    const int32_t block = table[at >> shift];
    const char* const from = paged_half(a.pages, it.kv_head, shift, block, at).k;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * (64 / kChunks) + lane / kChunks;
      load_shared<true>(from, r * a.pages.token + (lane % kChunks ^ Ring::k_turn(r)) * 16,
                  &held[wave][p * 16 * kChunks + i * 64]);
    }
    own_block = g % kParts == p ? block : own_block;
  }
  const OwnPlace own(a, it, begin + lane % kWavePlaces, own_block);
  const bool whole = seen_whole(a.sight, it.base, last, begin) &&
                     seen_whole(a.sight, it.base, last, begin + kWavePlaces - kTile);
  float w[kParts] = {};
#pragma unroll 1
  for (int32_t row = 0; row < it.rows; row += 16) {
    v8 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const v4u x = weigh_query8<T>(a, it, row + m, 32 * s + 8 * g);
      __builtin_memcpy(&q[s], &x, 16);
    }
    const float own_log = row_log(a, it, row + m);
    const int32_t own_position = it.base + quotient(min(row + m, it.rows - 1), a.group);
    // K is here (this wave alone reads what it asked for: none to meet)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    float log[4];
    int32_t position[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      log[i] = __shfl(own_log, 4 * g + i);
      position[i] = __shfl(own_position, 4 * g + i);
    }
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        v8 k;
        __builtin_memcpy(&k, &held[wave][p * 16 * kChunks + Ring::k_at(m, 4 * s + g)], 16);
        x = Matrix<T>::mma(q[s], k, x);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool sees = (log[i] != INFINITY) &
                          (whole | seen(a.sight, position[i], begin + 16 * p + m));
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.sight.c, -log[i]));
        w[p] += sees ? e : 0.f;
      }
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    w[p] += __shfl_xor(w[p], 16);
    w[p] += __shfl_xor(w[p], 32);
    sum = g == p ? w[p] : sum;
  }
  if (g < kParts) own.add(sum);
}

// Sum of a value over the 32 lanes of a wave's half, in all of them; by moves inside
// the vector unit (through shared memory 160 of them took 8 us).
template <int MOVE>
__device__ __forceinline__ float add_moved(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), MOVE, 0xF, 0xF,
                                                        true));
}
__device__ __forceinline__ float half_sum(float x) {
  x = add_moved<0xB1>(x);     // lanes 1, 0, 3, 2 of four
  x = add_moved<0x4E>(x);     // 2, 3, 0, 1
  x = add_moved<0x141>(x);    // eight lanes in the other order
  x = add_moved<0x140>(x);    // sixteen
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// More rows: S^T = K Q^T by 32 x 32 x 16. A wave holds 64 places of K, lane l's row is l %
// 32 of 32, and each lane adds up its own rows' shares, 32 sums, until the end: a row's
// log-sum-exp and position are its lane's, and no wave waits for another. The four waves of
// a workgroup share its places, each takes every fourth 32 rows; queries come straight from
// memory to shared memory of the wave's own, whole rows at a time and a step ahead. Bound by
// the vector unit (a score takes an exponential, a quarter of its rate, a product and a sum:
// 1.5 times its matrix products at 128 wide, 3 times at 64), busy 53 % of the time, and by
// the ends of few workgroups. The four prompts above, 128 wide: 128 to 135 us (585 to 617
// TFLOP/s); three chunks of 512 under 64-wide heads and a window of 4,096: 102. With four
// waves in step the prompts took 252; with exponentials beside the next part's products 135
// where they took 128.
constexpr int kRowsPlaces = 64, kRowsParts = kRowsPlaces / 32;

template <int D, typename T>
__global__ __launch_bounds__(kPagedLanes, D <= 64 ? 3 : D <= 128 ? 2 : 1)
void paged_weigh_rows_kernel(WeighArgs a) {
  typedef typename Matrix<T>::v8 v8;
  typedef PagedRing<D> Ring;
  constexpr int kSteps = D / 16, kShare = kWeighPlaces / kRowsPlaces;
  __shared__ v4u queue[kPagedWaves][2][32 * (D / 8)];
  __shared__ float side[kPagedWaves][kRowsPlaces];
  WeighItem it;
  const int32_t tile = blockIdx.x / (kShare * a.kv_heads);
  const int32_t rest = blockIdx.x - tile * kShare * a.kv_heads, share = rest / a.kv_heads;
  if (!find_places<true>(a, tile * a.kv_heads + rest - share * a.kv_heads, &it)) return;
  it.first += share * kRowsPlaces;
  if (!it.reaches(a.sight, it.first, kRowsPlaces)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, n = lane % 32, h = lane / 32;
  const auto* table = in_plan<int32_t>(a.plan, a.at_table) + it.table;
  const int32_t last = it.len - 1, shift = a.sight.block_shift;
  const int32_t group = static_cast<int32_t>(a.group.by);
  v8 k[kRowsParts][kSteps];
#pragma unroll
  for (int p = 0; p < kRowsParts; ++p) {
    const int32_t at = min(it.first + 32 * p + n, last);
    const char* from = paged_half(a.pages, it.kv_head, shift, table[at >> shift], at).k;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      load_bytes<16, false>(reinterpret_cast<uint32_t*>(&k[p][s]), from, 32 * s + 16 * h);
  }
  // rows that see a place of the workgroup's: from the first place on, and up to where the
  // window has left the last one
  const int32_t first_row = (max(0, it.first - it.base) * group) & ~31;
  int32_t end_row = it.rows;
  if (it.first >= a.sight.sinks && a.sight.window != INT32_MAX) {
    const int64_t end = (int64_t(it.first) + kRowsPlaces - 1 + a.sight.window - it.base) * group;
    end_row = static_cast<int32_t>(max<int64_t>(0, min<int64_t>(end_row, end)));
  }
  // 32 rows of queries come lane by lane as shared memory holds them (k_at). Where whole
  // tokens make 32 rows, and rows are aligned, a lane's place is the first row's and a fixed
  // distance; else each is looked up.
  constexpr int kStep = 32 * kPagedWaves, kChunks = D / 8, kLoads = 32 * kChunks / 64;
  const bool even = a.q.whole_words && 32 % group == 0 &&
                    max(a.q.token, a.q.head) < (1 << 24);     // 32-bit distances
  const T* const queries = reinterpret_cast<const T*>(a.q.base) + int64_t(it.token) * a.q.token +
                           int64_t(it.kv_head) * group * a.q.head;
  uint32_t place_of[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int slot = i * 64 + lane, r = slot / kChunks, at = slot % kChunks;
    const int32_t token = quotient(r, a.group);
    place_of[i] = static_cast<uint32_t>(
        (token * a.q.token + (r - token * group) * a.q.head) * 2 + (at ^ Ring::k_turn(r)) * 16);
  }
  const int32_t own_token = quotient(n, a.group);
  float next_log;
  int32_t next_token;
  const auto load = [&](int32_t row, v4u* to) {
    const int32_t first = __builtin_amdgcn_readfirstlane(quotient(row, a.group));
    if (even && row + 32 <= it.rows) {
      next_token = first + own_token;
      const char* const from = reinterpret_cast<const char*>(queries + first * a.q.token);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load_shared(from, place_of[i], to + 64 * i);
      next_log = a.lse[(int64_t(it.token) + next_token) * a.lse_token +
                       int64_t(it.kv_head) * group + (n - own_token * group)];
    } else {
      const int32_t own = min(row + n, it.rows - 1);
      next_token = quotient(own, a.group);
      next_log = a.lse[weigh_row(a, it, own, a.lse_token, 1)];
#pragma unroll 1
      for (int i = 0; i < kLoads; ++i) {
        const int slot = i * 64 + lane, r = slot / kChunks, at = slot % kChunks;
        to[slot] = weigh_query8<T>(a, it, row + r, 8 * (at ^ Ring::k_turn(r)));
      }
    }
  };
  int32_t row = first_row + 32 * wave;      // of the wave's first lane
  int turn = 0;
  f32x16 w[kRowsParts];
#pragma unroll
  for (int p = 0; p < kRowsParts; ++p) w[p] = f32x16{};
  if (row < end_row) load(row, queue[wave][0]);
  for (; row < end_row; row += kStep, turn ^= 1) {
    // what this wave asked for has come (it alone reads it: none to meet)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    v8 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      __builtin_memcpy(&q[s], &queue[wave][turn][Ring::k_at(n, 2 * s + h)], 16);
    const float log = row + n < it.rows ? 1.4426950408889634f * next_log : INFINITY;
    const int32_t position = it.base + next_token;
    if (row + kStep < end_row) load(row + kStep, queue[wave][turn ^ 1]);
    f32x16 x[kRowsParts];
#pragma unroll
    for (int p = 0; p < kRowsParts; ++p) x[p] = f32x16{};
#pragma unroll
    for (int p = 0; p < kRowsParts; ++p)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) x[p] = Matrix<T>::mma32(k[p][s], q[s], x[p]);
    const int32_t low = it.base + quotient(row, a.group);
    const int32_t high = it.base + quotient(min(row + 31, it.rows - 1), a.group);
#pragma unroll
    for (int p = 0; p < kRowsParts; ++p) {
      const int32_t place = it.first + 32 * p;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        x[p][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[p][i], a.sight.c, -log));
      if (!seen_whole(a.sight, low, high, place)) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          x[p][i] = seen(a.sight, position, place + 8 * (i / 4) + 4 * h + i % 4) ? x[p][i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) w[p][i] += x[p][i];
    }
  }
  // over the 32 lanes of a place, then over the waves
#pragma unroll
  for (int p = 0; p < kRowsParts; ++p)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float sum = half_sum(w[p][i]);
      if (n == 0) side[wave][32 * p + 8 * (i / 4) + 4 * h + i % 4] = sum;
    }
  __syncthreads();
  if (wave != 0) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPagedWaves; ++i) sum += side[i][lane];
  const int32_t place = it.first + lane;
  OwnPlace(a, it, place, table[min(place, last) >> shift]).add(sum);
}

// ---------------------------------------------------------------- eviction --

struct EvictArgs {
  const char* plan;
  const char* into_plan;        // the same: tokens stay in their blocks
  int64_t at_seqs, at_table, into_at_seqs, into_at_table;
  Pages pages;
  float* weights;               // [block][kv_head][token]
  int32_t* kept;                // [sequence][kv_head][keep]
  int64_t keep, sinks, recent;
  int64_t rows_each;            // move: of a workgroup
  int32_t groups;               // workgroups a sequence and head
  int32_t kv_heads, block_shift, row_chunks;   // 16-byte words of a row
};

constexpr int kSelectLanes = 1024, kSelectWaves = kSelectLanes / 64;

struct EvictSeq {
  int32_t len, kv_head;
  const AEGKV_CONSTANT int32_t* table;
  int64_t kept;                 // where its places are in `kept`
};

__device__ __forceinline__ EvictSeq evict_seq(const EvictArgs& a, int32_t index) {
  const int32_t s = index / a.kv_heads;
  const auto* seq = in_plan<Seq>(a.plan, a.at_seqs) + s;
  return EvictSeq{seq->len, index - s * a.kv_heads,
                  in_plan<int32_t>(a.plan, a.at_table) + seq->table, int64_t(index) * a.keep};
}

__device__ __forceinline__ int64_t weight_at(const EvictArgs& a,
                                             const AEGKV_CONSTANT int32_t* table, int32_t kv_head,
                                             int32_t place) {
  const int64_t block = table[place >> a.block_shift];
  return ((block * a.kv_heads + kv_head) << a.block_shift) +
         (place & ((1 << a.block_shift) - 1));
}

// Weights in the order of unsigned numbers; no number comes last.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);    // -0 is 0
  return u >> 31 ? ~u : u | 0x80000000u;
}

// What the waves before this one have written, added up by its lanes.
__device__ __forceinline__ uint32_t sum_before(const uint32_t (&of)[kSelectWaves], int wave,
                                               int lane) {
  uint32_t x = lane < wave ? of[lane] : 0;
#pragma unroll
  for (int far = 1; far < kSelectWaves; far *= 2) x += __shfl_xor(x, far);
  return __builtin_amdgcn_readfirstlane(x);
}

// Which places stay: the first `sinks`, the last `recent`, and of those between the
// ones of the largest weight, the earlier one of equals. The border weight is found
// eleven bits at a time from counts; then every wave goes through a run of places of its
// own, twice: once to count, once to write its places where they belong. STEPS: 64
// places each that a wave holds in registers from the first look on; 0: any number, read
// anew each time. A workgroup has a head's places to itself, so a long sequence is bound
// by what one compute unit does: five looks at a place, two to ten instructions each
// (30,001 places under 4 heads 21 us, 30 with a bound tested at every place; 48 x 8 heads
// of 1,500 to 8,000 places 16).
constexpr int kBins = 2048, kDigit = 11;
static_assert(kBins == 2 * kSelectLanes, "two bins a lane");

// How many lanes before this one are in `mask`.
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

template <int STEPS>
__global__ __launch_bounds__(kSelectLanes) void paged_select_kernel(EvictArgs a) {
  __shared__ uint32_t count[kBins], border, wanted;
  __shared__ uint32_t more[kSelectWaves], same[kSelectWaves];
  const EvictSeq e = evict_seq(a, blockIdx.x);
  int32_t* kept = a.kept + e.kept;
  if (e.len <= a.keep) {
    for (int64_t i = threadIdx.x; i < a.keep; i += kSelectLanes)
      kept[i] = i < e.len ? static_cast<int32_t>(i) : -1;
    return;
  }
  const int32_t keep = static_cast<int32_t>(a.keep), sinks = static_cast<int32_t>(a.sinks);
  const int32_t recent = static_cast<int32_t>(a.recent);
  for (int32_t i = threadIdx.x; i < sinks; i += kSelectLanes) kept[i] = i;
  for (int32_t i = threadIdx.x; i < recent; i += kSelectLanes)
    kept[keep - recent + i] = e.len - recent + i;
  const int32_t chosen = keep - sinks - recent, places = e.len - sinks - recent;
  if (chosen == 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  // places a wave goes through at a time
  constexpr int kAtOnce = STEPS ? 1 : 8, kTurn = 64 * kAtOnce;
  const int64_t run = (int64_t(places) - 1) / (kSelectWaves * kTurn) * kTurn + kTurn;
  const int32_t begin = static_cast<int32_t>(min(wave * run, int64_t(places)));
  const int32_t end = static_cast<int32_t>(min(int64_t(begin) + run, int64_t(places)));
  // a place behind the last one has the least key, and comes after all others of that key:
  // more than `chosen` are there, so it never stays
  const auto key = [&](int32_t i) {
    const uint32_t x =
        weight_key(a.weights[weight_at(a, e.table, e.kv_head, sinks + min(i, places - 1))]);
    return i < places ? x : 0;
  };
  // f(key, first place of the 64) for the wave's run
  uint32_t held[STEPS ? STEPS : 1];
  if constexpr (STEPS != 0) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) held[s] = key(begin + 64 * s + lane);
  }
  const auto each = [&](const auto& f) {
    if constexpr (STEPS != 0) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (begin + 64 * s >= end) break;
        f(held[s], begin + 64 * s);
      }
    } else {
      for (int32_t at = begin; at < end; at += 64 * kAtOnce) {
        uint32_t x[kAtOnce];
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s) x[s] = key(at + 64 * s + lane);
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s) f(x[s], at + 64 * s);
      }
    }
  };
  uint32_t prefix = 0, need = chosen;     // of the keys that share the bits found so far
#pragma unroll 1
  for (int shift = 32 - kDigit; ; shift = max(0, shift - kDigit)) {
    // the last digit, of the 32 bits' rest, is ten bits wide
    const int known = shift == 0 ? 10 : shift + kDigit;
    const bool first = shift == 32 - kDigit;
    for (int i = threadIdx.x; i < kBins; i += kSelectLanes) count[i] = 0;
    __syncthreads();
    const uint32_t mask = shift == 0 ? 1023u : kBins - 1;
    if (first)
      each([&](uint32_t x, int32_t) {
        atomicAdd(&count[x >> shift], 1u);
      });
    else
      each([&](uint32_t x, int32_t) {
        if (x >> known == prefix)
          atomicAdd(&count[x >> shift & mask], 1u);
      });
    __syncthreads();
    // a lane holds two neighbouring bins, the first lane the uppermost: bins above come
    // before
    const int low = kBins - 2 - 2 * static_cast<int>(threadIdx.x);
    const uint32_t upper = count[low + 1], lower = count[low];
    uint32_t before = upper + lower;
#pragma unroll
    for (int far = 1; far < 64; far *= 2) {
      const uint32_t x = __shfl_up(before, far);
      before += lane >= far ? x : 0;
    }
    if (lane == 63) more[wave] = before;
    __syncthreads();
    before += sum_before(more, wave, lane) - upper - lower;
    const bool in_upper = before < need && before + upper >= need;
    if (!in_upper) before += upper;
    if (in_upper || (before < need && before + lower >= need)) {
      const uint32_t bin = low + in_upper;
      border = first ? bin : prefix << (shift == 0 ? 10 : kDigit) | bin;
      wanted = need - before;
    }
    __syncthreads();
    prefix = border;
    need = wanted;
    if (shift == 0) break;
  }
  // now `prefix` is the border weight, of which the first `need` stay
  uint32_t above = 0, equal = 0;
  each([&](uint32_t x, int32_t) {
    above += x > prefix;
    equal += x == prefix;
  });
#pragma unroll
  for (int far = 1; far < 64; far *= 2) {
    above += __shfl_xor(above, far);
    equal += __shfl_xor(equal, far);
  }
  if (lane == 0) {
    more[wave] = above;
    same[wave] = equal;
  }
  __syncthreads();
  uint32_t equals = sum_before(same, wave, lane);
  int32_t* to = kept + sum_before(more, wave, lane) + sinks + min(equals, need);
  each([&](uint32_t x, int32_t at) {
    bool stays = x > prefix;
    const uint64_t same_here = __ballot(x == prefix);
    if (same_here) {
      stays |= (x == prefix) & (equals + lanes_below(same_here) < need);
      equals += __popcll(same_here);
    }
    const uint64_t all = __ballot(stays);
    if (stays) to[lanes_below(all)] = sinks + at + lane;
    to += __popcll(all);
  });
}

constexpr int kMoveLanes = 256, kMostMoveLanes = 1024, kMoveAtOnce = 8;

// Rows [r0, r1) of what stays, W at a time a lane's word of a row (`words` lanes a row).
// In their own blocks the rows go in order, and no row's place is taken before the rows
// that come with it and before it are read: row i comes from place kept[i] >= i, so
// later rows lie behind.
//
// Bound by HBM, whose rows of 256 bytes come in no order of theirs: 48 sequences of 1,500 to
// 8,000 tokens cut to 2,048, 8 KV heads of 128, take 158 us of 177 for both kernels (5.1
// TB/s). K, V and the weights of the same rows are neighbours, and their places come from
// the caches: with all of K first 168. A workgroup that moves K and V of a row at once
// takes longer (201 of both). In their own blocks one workgroup has all of a head's rows:
// of 1,024 lanes, since it waits for each turn (30,001 tokens to 4,096, 4 heads: 52 to 56 us
// of both kernels, 71 with 256 lanes).
template <typename W, typename F>
__device__ __forceinline__ void move_rows(const int32_t* kept, int64_t r0, int64_t r1,
                                          int words, bool in_place, const F& place) {
  const int lanes_row = words, rows = blockDim.x / lanes_row;
  const int row = threadIdx.x / lanes_row, word = threadIdx.x % lanes_row;
  for (int64_t i0 = r0; i0 < r1; i0 += rows * kMoveAtOnce) {
    W x[kMoveAtOnce];
    W* to[kMoveAtOnce];
#pragma unroll
    for (int u = 0; u < kMoveAtOnce; ++u) {
      const int64_t i = min(i0 + u * rows + row, r1 - 1);
      x[u] = *(place(false, kept[i]) + word);
      to[u] = place(true, static_cast<int32_t>(i)) + word;
    }
    if (in_place) __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveAtOnce; ++u)
      if (i0 + u * rows + row < r1) __builtin_nontemporal_store(x[u], to[u]);
  }
}

__global__ __launch_bounds__(kMostMoveLanes) void paged_move_kernel(EvictArgs a) {
  const int32_t which = blockIdx.x % 3, rest = blockIdx.x / 3;     // K, V or the weights
  const int32_t index = rest / a.groups, part = rest - index * a.groups;
  const EvictSeq e = evict_seq(a, index);
  const bool in_place = a.plan == a.into_plan;
  if (in_place && e.len <= a.keep) return;
  const int64_t rows = min(int64_t(e.len), a.keep);
  const int64_t r0 = part * a.rows_each, r1 = min(rows, r0 + a.rows_each);
  if (r0 >= r1) return;
  const auto* into = in_plan<int32_t>(a.into_plan, a.into_at_table) +
                     (in_plan<Seq>(a.into_plan, a.into_at_seqs) + index / a.kv_heads)->table;
  const int32_t* kept = a.kept + e.kept;
  if (which == 2) {
    move_rows<float>(kept, r0, r1, 1, in_place, [&](bool to, int32_t place) {
      return a.weights + weight_at(a, to ? into : e.table, e.kv_head, place);
    });
    return;
  }
  char* pages = const_cast<char*>(which ? a.pages.v : a.pages.k);
  const int64_t block = which ? a.pages.v_block : a.pages.k_block;
  move_rows<v4u>(kept, r0, r1, a.row_chunks, in_place, [&](bool to, int32_t place) {
    const int64_t id = (to ? into : e.table)[place >> a.block_shift];
    return reinterpret_cast<v4u*>(
        pages + id * block + int64_t(place & ((1 << a.block_shift) - 1)) * a.pages.token +
        int64_t(e.kv_head) * a.pages.head);
  });
}

}  // namespace

#endif  // AEGKV_PAGED_CACHE_H
