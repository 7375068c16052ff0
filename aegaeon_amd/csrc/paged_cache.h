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

// ---------------------------------------------------------- rotate, write --

// Where the values of a kind of heads come from and go to.
struct HeadRows {
  Values from, to;
  int32_t heads;
};

struct PlaceArgs {
  const char* plan;           // null: tokens are rows, one after another
  int64_t at_new_spans;
  int64_t tokens;             // without a plan
  int32_t chunk;              // tokens of a span without a plan
  const double* turns;        // a position's turns, for each pair
  const void* positions;      // null: the plan's
  int32_t position_bytes;
  int32_t pairs, interleaved;
  float amplitude;
  int32_t head_dim;
  HeadRows q, k;              // rotated
  Values v;                   // written as they are
  Pages pages;                // where k and v go (k.to: without a plan)
  int32_t kv_heads, block_shift;
  int32_t heads, heads_each, head_groups;   // of all kinds; of a workgroup; workgroups a span
};

constexpr int kPlaceLanes = 256;
constexpr int kPlaceTokens = 16;    // of a workgroup
constexpr int kMostAngles = kPlaceTokens * 128;

// N values as float32 and back, N = 1 or 8.
template <int N, typename T>
__device__ __forceinline__ void take(const T* p, bool whole_words, float* x) {
  if constexpr (N == 8) load8(p, whole_words, x);
  else x[0] = static_cast<float>(*p);
}
template <int N, typename T>
__device__ __forceinline__ void give(T* p, bool whole_words, const float* x) {
  if constexpr (N == 8) store8(p, whole_words, x);
  else *p = static_cast<T>(x[0]);
}

// (a, b) -> (a c - b s, b c + a s) for each pair, c and s the cosine and sine of
// position * turns: the angle in 64 bits, of which the whole turns are dropped before
// it is rounded (positions of millions keep their angle), values in 32, one
// rounding at the end. A workgroup takes up to 16 tokens of some heads: the angles,
// 60 instructions each, are made once for all of them.
// G: type of k and v; T: of q, of what is written and of what comes of q. N: pairs of
// an item. A lane takes 2 N values of a head at once: N at a and N at b.
template <int N, typename G, typename T>
__global__ __launch_bounds__(kPlaceLanes) void place_rows_kernel(PlaceArgs a) {
  __shared__ float cosine[kMostAngles], sine[kMostAngles];
  const int32_t span = blockIdx.x / a.head_groups;
  const int32_t first_head = (blockIdx.x - span * a.head_groups) * a.heads_each;
  const int32_t heads = min(a.heads_each, a.heads - first_head);
  int64_t token;
  int32_t count, position = 0, block = 0, inside = 0;
  if (a.plan) {
    if (span >= in_plan<Header>(a.plan, 0)->new_spans) return;
    const auto* s = in_plan<NewSpan>(a.plan, a.at_new_spans) + span;
    token = s->token;
    count = s->count;
    position = s->position;
    block = s->block;
    inside = s->inside;
  } else {
    token = int64_t(span) * a.chunk;
    count = static_cast<int32_t>(min<int64_t>(a.chunk, a.tokens - token));
  }
  // (v's heads need no angles)
  if (first_head < a.q.heads + a.k.heads) {
    for (int32_t i = threadIdx.x; i < count * a.pairs; i += kPlaceLanes) {
      const int32_t t = i / a.pairs, pair = i - t * a.pairs;
      int64_t p = position + t;
      if (a.positions)
        p = a.position_bytes == 8 ? static_cast<const int64_t*>(a.positions)[token + t]
                                  : static_cast<const int32_t*>(a.positions)[token + t];
      double turn = static_cast<double>(p) * a.turns[pair];
      turn -= rint(turn);
      float s, c;
      sincospif(static_cast<float>(2 * turn), &s, &c);
      cosine[i] = c * a.amplitude;
      sine[i] = s * a.amplitude;
    }
  }
  __syncthreads();
  const int32_t units = a.head_dim / (2 * N), turned = a.pairs / N;
  const int32_t items = count * heads * units;
  const int64_t k_at = a.plan ? block * a.pages.k_block : 0;
  const int64_t v_at = a.plan ? block * a.pages.v_block : 0;
#pragma unroll 2
  for (int32_t i = threadIdx.x; i < items; i += kPlaceLanes) {
    const int32_t row = i / units, u = i - row * units;
    const int32_t t = row / heads;
    int32_t head = first_head + row - t * heads;
    int32_t at = 2 * N * u, next = at + N;      // untouched values, interleaved pairs
    const bool turn = u < turned && head < a.q.heads + a.k.heads;
    if (turn && !a.interleaved) {
      at = N * u;
      next = at + a.pairs;
    }
    const auto work = [&](const auto* from, bool from_words, auto* to, bool to_words) {
      float x[N], y[N];
      take<N>(from + at, from_words, x);
      take<N>(from + next, from_words, y);
      if (turn) {
        const float* c = cosine + t * a.pairs + N * u;
        const float* s = sine + t * a.pairs + N * u;
        if (!a.interleaved || N == 1) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float p = x[j] * c[j] - y[j] * s[j];
            y[j] = y[j] * c[j] + x[j] * s[j];
            x[j] = p;
          }
        } else {
          const auto spin = [&](float* z, const float* cc, const float* ss) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
              const float p = z[2 * j] * cc[j] - z[2 * j + 1] * ss[j];
              z[2 * j + 1] = z[2 * j + 1] * cc[j] + z[2 * j] * ss[j];
              z[2 * j] = p;
            }
          };
          spin(x, c, s);
          spin(y, c + N / 2, s + N / 2);
        }
      }
      give<N>(to + at, to_words, x);
      give<N>(to + next, to_words, y);
    };
    const int64_t r = token + t;
    if (head < a.q.heads) {
      const Values f = a.q.from, o = a.q.to;
      work(reinterpret_cast<const T*>(f.base) + r * f.token + head * f.head, f.whole_words,
           reinterpret_cast<T*>(o.base) + r * o.token + head * o.head, o.whole_words);
      continue;
    }
    head -= a.q.heads;
    const bool key = head < a.k.heads;
    if (!key) head -= a.k.heads;
    const Values f = key ? a.k.from : a.v;
    const G* from = reinterpret_cast<const G*>(f.base) + r * f.token + head * f.head;
    if (a.plan) {
      char* page = const_cast<char*>(key ? a.pages.k + k_at : a.pages.v + v_at);
      work(from, f.whole_words,
           reinterpret_cast<T*>(page + int64_t(inside + t) * a.pages.token +
                                int64_t(head) * a.pages.head), true);
    } else {
      const Values o = a.k.to;
      work(from, f.whole_words, reinterpret_cast<G*>(o.base) + r * o.token + head * o.head,
           o.whole_words);
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

// log2 of what sums are taken against: exactly what the exponents had added.
template <typename T>
__device__ __forceinline__ float row_base(const RowSum& s, float c) {
  return fabsf(s.lift) > Matrix<T>::kLimit && s.top != -INFINITY ? s.top * c - Matrix<T>::kLift
                                                                 : -s.lift;
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

// Whether one of a word's two values is an infinity or no number.
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t kExponent = std::is_same<T, __bf16>::value ? 0x7F80u : 0x7C00u;
  return (w & kExponent) == kExponent || ((w >> 16) & kExponent) == kExponent;
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
// byte permutes.
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
        load_bytes<16, true>(reinterpret_cast<uint32_t*>(&k[i][s]), h[i].k,
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
        bool bad = false;
#pragma unroll
        for (int w = 0; w < kWords; ++w) bad |= not_finite<T>(v[half][t][w]);
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
                 16 * (t % 16 / 4) + m));
      weight[r] = static_cast<float>(
          __builtin_bit_cast(T, static_cast<uint16_t>(t % 2 ? pair >> 16 : pair)));
      sees[r] = seen(a, position[r], j);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int run = 4 * g + i;
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
// A stage of 64 tokens' K and V lies in shared memory as rows of 16-byte chunks, each
// row's chunks exchanged by its number so that neither product's reads meet in a bank:
// K's operands are a token's chunk a lane, V's come four tokens of a value a lane by
// transposing reads. Lane l (row l % 32, h = l / 32) holds the scores of tokens 8 (i / 4)
// + 4 h + i % 4, i < 16, and they are the second product's operand as they lie.
constexpr int kStageTokens = 64, kRowsWave = 32;
static_assert(kManyRows == kPagedWaves * kRowsWave, "rows of a workgroup");

template <int D>
struct PagedStage {
  static constexpr int kChunks = D / 8;    // of 16 bytes in a row
  v4u k[kStageTokens * kChunks];
  v4u v[kStageTokens * kChunks];
  static __device__ __forceinline__ int k_at(int token, int chunk) {
    return token * kChunks + (chunk ^ (D == 64 ? token / 2 % 8 : token % 16));
  }
  static __device__ __forceinline__ int v_at(int token, int chunk) {
    return token * kChunks + (chunk ^ (2 * (token % 4)));
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Of 16 lanes that point at four rows of 16 values, four values a lane: lane i gets
// value i of the four rows.
__device__ __forceinline__ s16x4 read_turned(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
}

template <int D, typename T>
__device__ __forceinline__ void paged_prompt_item(const Sight& a, const Pages& pages,
                                                  PagedItem it, PagedStage<D> (&stages)[2]) {
  typedef typename Matrix<T>::v8 v8;
  typedef PagedStage<D> Stage;
  constexpr int kSteps = D / 16, kOut = D / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, n = lane % 32, h = lane / 32;
  const PagedCold args = paged_cold();
  const auto* table = in_plan<int32_t>(args->plan, args->at_table) + it->table;
  const Tiles tiles = {it->first_tiles, it->window_tile - it->first_tiles, it->tile_end};
  const int32_t group = args->group, kv_head = it->kv_head;

  // this wave's share of a stage: 16 tokens, kRows of them at a time
  constexpr int kLanesRow = Stage::kChunks < 64 ? Stage::kChunks : 64;
  constexpr int kRows = 64 / kLanesRow, kLoads = 16 / kRows;
  const int own_tile = wave / 2, own_half = wave % 2;
  const int load_row = lane / kLanesRow, load_chunk = lane % kLanesRow;
  v4u held_k[kLoads], held_v[kLoads];
  const auto load = [&](int32_t at) {
    // behind the last tile the last one is read again, and not used
    const int32_t position = tiles.at(min(at + own_tile, tiles.end - 1)) * kTile + 16 * own_half;
    const PagedHalf half = paged_half(pages, kv_head, a.block_shift,
                                      table[position >> a.block_shift], position);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t offset = (i * kRows + load_row) * pages.token + load_chunk * 16;
      load_bytes<16, false>(reinterpret_cast<uint32_t*>(&held_k[i]), half.k, offset);
      load_bytes<16, false>(reinterpret_cast<uint32_t*>(&held_v[i]), half.v, offset);
    }
  };
  const auto lay = [&](Stage& to) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int token = 16 * wave + i * kRows + load_row;
      to.k[Stage::k_at(token, load_chunk)] = held_k[i];
      to.v[Stage::v_at(token, load_chunk)] = held_v[i];
    }
  };
  load(it->tile);

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
  f32x16 o[kOut];
#pragma unroll
  for (int d = 0; d < kOut; ++d) o[d] = f32x16{};
  RowSum state;

  // where a lane reads V turned: token (lane % 16) / 4 of four, 4 values of 16
  const int turn_token = lane % 16 / 4, turn_chunk = 2 * (lane / 16 % 2) + lane % 4 / 2;

  const auto multiply = [&](const Stage& from, int32_t at, int tile) {
    if (at + tile >= tiles.end) return;
    const int32_t begin = tiles.at(at + tile) * kTile;
    // tiles that none of the wave's rows sees
    if ((begin > high) | ((low - (begin + kTile - 1) >= a.window) & (begin >= a.sinks))) return;
    f32x16 x = {};
    v8 k[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      __builtin_memcpy(&k[s], &from.k[Stage::k_at(32 * tile + n, 2 * s + h)], 16);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) x = Matrix<T>::mma32(k[s], q[s], x);
    // V: tokens 16 ks + 4 h + j and 16 ks + 8 + 4 h + j of a value
    uint32_t v[2][kOut][4];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int d = 0; d < kOut; ++d)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int token = 32 * tile + 16 * ks + 8 * j + 4 * h + turn_token;
          const s16x4 y = read_turned(
              reinterpret_cast<const char*>(&from.v[Stage::v_at(token, 4 * d + turn_chunk)]) +
              8 * (lane % 2));
          __builtin_memcpy(&v[ks][d][2 * j], &y, 8);
        }
    float e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = x[i];
    const bool whole = seen_whole(a, low, high, begin);
    const auto some_sees = [&](int32_t j) {
      return (j <= high) & ((low - j < a.window) | (j < a.sinks));
    };
    bool odd = false;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        e[i] = seen(a, position, begin + 8 * (i / 4) + 4 * h + i % 4) ? e[i] : -INFINITY;
      // infinities and no numbers: a probability of 0 would make no number of them
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t bad = (not_finite<T>(v[ks][d][w] & 0xFFFFu) ? 0xFFFFu : 0u) |
                                 (not_finite<T>(v[ks][d][w] & 0xFFFF0000u) ? 0xFFFF0000u : 0u);
            const int32_t j = begin + 16 * ks + 8 * (w / 2) + 4 * h + 2 * (w % 2);
            odd |= ((bad & 0xFFFFu) && some_sees(j)) || ((bad >> 16) && some_sees(j + 1));
            v[ks][d][w] &= ~bad;
          }
    }
    softmax_part<T>(e, a.c, state, o, [](float y) { return pair_max(y); });
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const v8 p = round8<T>(e, 8 * ks);
#pragma unroll
      for (int d = 0; d < kOut; ++d) {
        v8 y;
        __builtin_memcpy(&y, v[ks][d], 16);
        o[d] = Matrix<T>::mma32(y, p, o[d]);
      }
    }
    if (!whole && __any(odd)) {
      // what was taken out goes to the rows that see its token
#pragma unroll 1
      for (int t = 0; t < kTile; ++t) {
        const int32_t j = begin + t;
        const bool sees = seen(a, position, j);
        // the row's probability of token t, from the lane that has it
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          mine = i == 4 * (t / 8) + t % 4 ? static_cast<float>(static_cast<T>(e[i])) : mine;
        const float weight = __shfl(mine, n + 32 * (t / 4 % 2));
#pragma unroll
        for (int d = 0; d < kOut; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int value = 32 * d + 8 * (i / 4) + 4 * h + i % 4;
            const T y = reinterpret_cast<const T*>(
                &from.v[Stage::v_at(32 * tile + t, value / 8)])[value % 8];
            const bool bad = not_finite<T>(__builtin_bit_cast(uint16_t, y));
            const float was = o[d][i];
            o[d][i] = (bad & sees) ? __builtin_fmaf(weight, static_cast<float>(y), was) : was;
          }
      }
    }
  };

  int turn = 0;
  for (int32_t at = it->tile; at < tiles.end; at += 2, turn ^= 1) {
    lay(stages[turn]);
    load(at + 2);
    __syncthreads();
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) multiply(stages[turn], at, tile);
  }

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
      const int first = 32 * d + 8 * i + 4 * h;
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = o[d][4 * i + j] * inv;
      if (slot >= 0) {
        __builtin_memcpy(part + first, y, 16);
      } else {
        T t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = static_cast<T>(y[j]);
        if (end_args->out.whole_words) {
          __builtin_memcpy(__builtin_assume_aligned(to + first, 8), t, 8);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) to[first + j] = t[j];
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
  __shared__ PagedStage<D> stages[2];
  const Sight sight = args.sight;
  const Pages pages = args.pages;
  const PagedItem it = in_plan<Item>(args.plan, args.at_items) + blockIdx.x;
  if (static_cast<int32_t>(blockIdx.x) >= in_plan<Header>(args.plan, 0)->items[args.kind]) return;
  paged_prompt_item<D, T>(sight, pages, it, stages);
}

// Rows whose tiles several items shared: their parts, scaled to the largest base of
// all, over the sum of their sums. A workgroup's lanes are groups of D / 4,
// four values a lane. Of up to kMergeRows parts each group takes rows of its own;
// more (few rows over a long axis) are shared out to the groups, one row a workgroup.
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
  int64_t at_seqs, at_table;
  Values q;
  const float* lse;
  int64_t lse_token;
  float* weights;       // [block][kv_head][token]
  int32_t group, kv_heads;
};

// Places of a workgroup, and of one of its waves.
constexpr int kWeighPlaces = kPlaceTile, kWavePlaces = kWeighPlaces / kPagedWaves;

// One workgroup's work: places of one sequence under one KV head, and its queries.
struct WeighItem {
  int32_t kv_head, first;               // of the places
  int32_t len, base, rows, token, table;
  // Whether some query sees a place of [from, from + count).
  __device__ __forceinline__ bool reaches(const Sight& a, int32_t from, int32_t count) const {
    return (from < len) & ((base - (from + count - 1) < a.window) | (from < a.sinks));
  }
};

__device__ __forceinline__ bool find_places(const WeighArgs& a, WeighItem* it) {
  const int32_t i = blockIdx.x / a.kv_heads;
  const auto* h = in_plan<Header>(a.plan, 0);
  if (i >= h->place_tiles) return false;
  const auto* seq = in_plan<Seq>(a.plan, a.at_seqs);
  // the last sequence that begins at or before tile i; empty sequences begin where the
  // next one does
  int32_t lo = 0, hi = h->num_seqs - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) >> 1;
    if (seq[mid].place_tile <= i) lo = mid;
    else hi = mid - 1;
  }
  const auto* s = seq + lo;
  it->kv_head = blockIdx.x - i * a.kv_heads;
  it->first = (i - s->place_tile) * kWeighPlaces;
  it->len = s->len;
  it->base = s->len - s->fresh;
  it->rows = s->fresh * a.group;
  it->token = s->token;
  it->table = s->table;
  return it->rows > 0;
}

// Eight values of a query row from `at` on; 0 where there is none.
template <typename T>
__device__ __forceinline__ v4u weigh_query8(const WeighArgs& a, const WeighItem& it, int32_t row,
                                            int32_t at) {
  v4u x = {0, 0, 0, 0};
  if (row < it.rows) {
    const int32_t token = row / a.group;
    const T* from = reinterpret_cast<const T*>(a.q.base) +
                    (int64_t(it.token) + token) * a.q.token +
                    (int64_t(it.kv_head) * a.group + (row - token * a.group)) * a.q.head + at;
    if (a.q.whole_words) {
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

// log2(e) times a row's log-sum-exp; infinity where there is no row: its share is 0.
__device__ __forceinline__ float row_log(const WeighArgs& a, const WeighItem& it, int32_t row) {
  if (row >= it.rows) return INFINITY;
  const int32_t token = row / a.group;
  return 1.4426950408889634f * a.lse[(int64_t(it.token) + token) * a.lse_token +
                                     int64_t(it.kv_head) * a.group + (row - token * a.group)];
}

__device__ __forceinline__ void add_weight(const WeighArgs& a, const WeighItem& it,
                                           const AEGKV_CONSTANT int32_t* table, int32_t place,
                                           float w) {
  if (!it.reaches(a.sight, place, 1)) return;
  const int32_t shift = a.sight.block_shift;
  const int64_t block = table[place >> shift];
  float* to = a.weights + (((block * a.kv_heads + it.kv_head) << shift) +
                           (place & ((1 << shift) - 1)));
  *to = (place < it.base ? *to : 0.f) + w;
}

// w[place] += sum over the rows that see it of exp2(c s - log2(e) lse). A place
// belongs to one lane at the end: no atomics, and the sum's order is fixed. Up
// to 64 rows of a sequence: S = Q K^T by 16 x 16 x 32, a wave's 64 places in registers.
template <int D, typename T>
__global__ __launch_bounds__(kPagedLanes, D <= 128 ? 3 : 2) void paged_weigh_kernel(WeighArgs a) {
  typedef typename Matrix<T>::v8 v8;
  constexpr int kSteps = D / 32, kParts = kWavePlaces / 16;
  WeighItem it;
  if (!find_places(a, &it) || it.rows > kMostMore) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, m = lane % 16, g = lane / 16;
  const int32_t begin = it.first + wave * kWavePlaces;
  if (!it.reaches(a.sight, begin, kWavePlaces)) return;
  const auto* table = in_plan<int32_t>(a.plan, a.at_table) + it.table;
  const int32_t last = it.len - 1, shift = a.sight.block_shift;
  v8 k[kParts][kSteps];
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    // (parts behind the sequence's last place read its last one again)
    const int32_t at = min(begin + 16 * p, last & ~15);
    const PagedHalf h = paged_half(a.pages, it.kv_head, shift, table[at >> shift], at);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      load_bytes<16, true>(reinterpret_cast<uint32_t*>(&k[p][s]), h.k,
                           m * a.pages.token + g * 16 + s * 64);
  }
  float w[kParts] = {};
#pragma unroll 1
  for (int32_t row = 0; row < it.rows; row += 16) {
    v8 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const v4u x = weigh_query8<T>(a, it, row + m, 32 * s + 8 * g);
      __builtin_memcpy(&q[s], &x, 16);
    }
    float log[4];
    int32_t position[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      log[i] = row_log(a, it, row + 4 * g + i);
      position[i] = it.base + min(row + 4 * g + i, it.rows - 1) / a.group;
    }
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) x = Matrix<T>::mma(q[s], k[p][s], x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.sight.c, -log[i]));
        const bool sees = (row + 4 * g + i < it.rows) &
                          seen(a.sight, position[i], begin + 16 * p + m);
        w[p] += sees ? e : 0.f;
      }
    }
  }
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    w[p] += __shfl_xor(w[p], 16);
    w[p] += __shfl_xor(w[p], 32);
    if (g == p) add_weight(a, it, table, begin + 16 * p + m, w[p]);
  }
}

// More rows: S by 32 x 32 x 16, the rows' queries in shared memory for all four
// waves, 32 rows a stage, two stages.
template <int D>
struct WeighStage {
  v4u q[32 * (D / 8)];
  float log[32];
  int32_t position[32];
};

template <int D, typename T>
__global__ __launch_bounds__(kPagedLanes, D <= 128 ? 2 : 1) void paged_weigh_rows_kernel(
    WeighArgs a) {
  typedef typename Matrix<T>::v8 v8;
  typedef PagedStage<D> Place;
  constexpr int kSteps = D / 16, kParts = kWavePlaces / 32, kChunks = D / 8;
  __shared__ WeighStage<D> stages[2];
  WeighItem it;
  if (!find_places(a, &it) || it.rows <= kMostMore) return;
  if (!it.reaches(a.sight, it.first, kWeighPlaces)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, n = lane % 32, h = lane / 32;
  const int32_t begin = it.first + wave * kWavePlaces;
  const auto* table = in_plan<int32_t>(a.plan, a.at_table) + it.table;
  const int32_t last = it.len - 1, shift = a.sight.block_shift;
  v8 k[kParts][kSteps];
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    const int32_t at = min(begin + 32 * p + n, last);
    const char* from = paged_half(a.pages, it.kv_head, shift, table[at >> shift], at).k;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      load_bytes<16, false>(reinterpret_cast<uint32_t*>(&k[p][s]), from, 32 * s + 16 * h);
  }
  // rows that see a place of the workgroup's: from the first place on, and up to where the
  // window has left the last one
  const int32_t first_row = max(0, it.first - it.base) * a.group & ~31;
  int32_t end_row = it.rows;
  if (it.first >= a.sight.sinks && a.sight.window != INT32_MAX) {
    const int64_t end = (int64_t(it.first) + kWeighPlaces - 1 + a.sight.window - it.base) *
                        a.group;
    end_row = static_cast<int32_t>(max<int64_t>(0, min<int64_t>(end_row, end)));
  }
  constexpr int kLoads = 32 * kChunks / kPagedLanes;
  v4u held[kLoads];
  float held_log = 0.f;
  const auto load = [&](int32_t row) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * kPagedLanes + threadIdx.x;
      held[i] = weigh_query8<T>(a, it, row + at / kChunks, at % kChunks * 8);
    }
    if (threadIdx.x < 32) held_log = row_log(a, it, row + threadIdx.x);
  };
  load(first_row);
  float w[kParts] = {};
  int turn = 0;
  for (int32_t row = first_row; row < end_row; row += 32, turn ^= 1) {
    WeighStage<D>& stage = stages[turn];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * kPagedLanes + threadIdx.x;
      stage.q[Place::k_at(at / kChunks, at % kChunks)] = held[i];
    }
    if (threadIdx.x < 32) {
      stage.log[threadIdx.x] = held_log;
      stage.position[threadIdx.x] =
          it.base + min(row + static_cast<int32_t>(threadIdx.x), it.rows - 1) / a.group;
    }
    load(row + 32);
    __syncthreads();
    const int32_t low = stage.position[0], high = stage.position[31];
    v8 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      __builtin_memcpy(&q[s], &stage.q[Place::k_at(n, 2 * s + h)], 16);
    float log[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) log[i] = stage.log[8 * (i / 4) + 4 * h + i % 4];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const int32_t place = begin + 32 * p;
      f32x16 x = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) x = Matrix<T>::mma32(q[s], k[p][s], x);
      float e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.sight.c, -log[i]));
      if (!seen_whole(a.sight, low, high, place) || row + 32 > it.rows) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = 8 * (i / 4) + 4 * h + i % 4;
          const bool sees = (row + r < it.rows) & seen(a.sight, stage.position[r], place + n);
          e[i] = sees ? e[i] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) w[p] += e[i];
    }
  }
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    w[p] += __shfl_xor(w[p], 32);
    if (h == p) add_weight(a, it, table, begin + 32 * p + n, w[p]);
  }
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

// Which places stay: the first `sinks`, the last `recent`, and of those between the
// ones of the largest weight, the earlier one of equals. The border weight is found
// eight bits at a time from counts; then every wave goes through a run of its own, twice:
// once to count, once to write its places where they belong.
__global__ __launch_bounds__(kSelectLanes) void paged_select_kernel(EvictArgs a) {
  __shared__ uint32_t count[256], border, wanted;
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
  const auto key = [&](int32_t i) {
    return weight_key(a.weights[weight_at(a, e.table, e.kv_head, sinks + i)]);
  };
  uint32_t prefix = 0, need = chosen;     // of the keys that share the bits found so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) count[threadIdx.x] = 0;
    __syncthreads();
    for (int32_t i = threadIdx.x; i < places; i += kSelectLanes) {
      const uint32_t x = key(i);
      if (shift == 24 || x >> (shift + 8) == prefix)
        atomicAdd(&count[x >> shift & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
      // lane l holds the four bins from 252 - 4 l on: bins above it come before it
      const int top = 252 - 4 * static_cast<int>(threadIdx.x);
      uint32_t mine[4], all = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) all += mine[i] = count[top + i];
      uint32_t before = all;
#pragma unroll
      for (int far = 1; far < 64; far *= 2) {
        const uint32_t x = __shfl_up(before, far);
        before += static_cast<int>(threadIdx.x) >= far ? x : 0;
      }
      before -= all;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        if (before < need && before + mine[i] >= need) {
          border = prefix << 8 | static_cast<uint32_t>(top + i);
          wanted = need - before;
        }
        before += mine[i];
      }
    }
    __syncthreads();
    prefix = border;
    need = wanted;
  }
  // now `prefix` is the border weight, of which the first `need` stay
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int32_t run = ((places + kSelectWaves - 1) / kSelectWaves + 63) & ~63;
  const int32_t begin = min(int64_t(wave) * run, int64_t(places));
  const int32_t end = min(int64_t(begin) + run, int64_t(places));
  uint32_t above = 0, equal = 0;
  for (int32_t i = begin; i < end; i += 64) {
    const uint32_t x = i + lane < end ? key(i + lane) : 0;
    const bool there = i + lane < end;
    above += __popcll(__ballot(there && x > prefix));
    equal += __popcll(__ballot(there && x == prefix));
  }
  if (lane == 0) {
    more[wave] = above;
    same[wave] = equal;
  }
  __syncthreads();
  uint32_t to = 0, equals = 0;
  for (int w = 0; w < wave; ++w) {
    to += more[w];
    equals += same[w];
  }
  to += sinks + min(equals, need);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  for (int32_t i = begin; i < end; i += 64) {
    const bool there = i + lane < end;
    const uint32_t x = there ? key(i + lane) : 0;
    const bool is_equal = there && x == prefix;
    const uint64_t same_here = __ballot(is_equal);
    const bool stays = (there && x > prefix) ||
                       (is_equal && equals + __popcll(same_here & below) < need);
    const uint64_t all = __ballot(stays);
    if (stays) kept[to + __popcll(all & below)] = sinks + i + lane;
    to += __popcll(all);
    equals += __popcll(same_here);
  }
}

constexpr int kMoveLanes = 256, kMoveAtOnce = 8;

// Rows [r0, r1) of what stays, W at a time a lane's word of a row (`words` lanes a row).
// In their own blocks the rows go in order, and no row's place is taken before the rows
// that come with it and before it are read: row i comes from place kept[i] >= i, so
// later rows lie behind.
template <typename W, typename F>
__device__ __forceinline__ void move_rows(const int32_t* kept, int64_t r0, int64_t r1,
                                          int words, bool in_place, const F& place) {
  const int lanes_row = words, rows = kMoveLanes / lanes_row;
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
      if (i0 + u * rows + row < r1) *to[u] = x[u];
  }
}

__global__ __launch_bounds__(kMoveLanes) void paged_move_kernel(EvictArgs a) {
  const int32_t index = blockIdx.x / a.groups, part = blockIdx.x - index * a.groups;
  const EvictSeq e = evict_seq(a, index);
  const bool in_place = a.plan == a.into_plan;
  if (in_place && e.len <= a.keep) return;
  const int64_t rows = min(int64_t(e.len), a.keep);
  const int64_t r0 = part * a.rows_each, r1 = min(rows, r0 + a.rows_each);
  if (r0 >= r1) return;
  const auto* into = in_plan<int32_t>(a.into_plan, a.into_at_table) +
                     (in_plan<Seq>(a.into_plan, a.into_at_seqs) + index / a.kv_heads)->table;
  const int32_t* kept = a.kept + e.kept;
  if (blockIdx.y == 2) {
    move_rows<float>(kept, r0, r1, 1, in_place, [&](bool to, int32_t place) {
      return a.weights + weight_at(a, to ? into : e.table, e.kv_head, place);
    });
    return;
  }
  char* pages = const_cast<char*>(blockIdx.y ? a.pages.v : a.pages.k);
  const int64_t block = blockIdx.y ? a.pages.v_block : a.pages.k_block;
  move_rows<v4u>(kept, r0, r1, a.row_chunks, in_place, [&](bool to, int32_t place) {
    const int64_t id = (to ? into : e.table)[place >> a.block_shift];
    return reinterpret_cast<v4u*>(
        pages + id * block + int64_t(place & ((1 << a.block_shift) - 1)) * a.pages.token +
        int64_t(e.kv_head) * a.pages.head);
  });
}

}  // namespace

#endif  // AEGKV_PAGED_CACHE_H
