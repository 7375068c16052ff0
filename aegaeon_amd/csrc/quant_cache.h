// A quantised paged KV cache: kernels that write tokens into it, read them back
// and attend over it. Part of aegkv.hip's translation unit, whose checks of
// device memory and error texts it uses; contracts are in include/aegkv.h.
//
// Format of a page (one block of K or of V): kv_heads chunks, one a head. A
// chunk is block_size rows of codes, then for each group of 32 values of the
// head a plane of block_size scale bytes. Codes and scales of one head lie
// together so that attention, which takes a head at a time, reads whole lines.
#ifndef AEGKV_QUANT_CACHE_H
#define AEGKV_QUANT_CACHE_H

#include "batch_plan.h"

namespace {

using namespace aegkv_batch;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

template <int FMT>
struct Format;
template <>
struct Format<AEGKV_FORMAT_MXFP4> {
  static constexpr int kBits = 4;
  static constexpr uint32_t kCarry = 0x3FFFFF, kTop = 2;  // largest value 1.5 * 2^2
};
template <>
struct Format<AEGKV_FORMAT_MXFP8> {
  static constexpr int kBits = 8;
  static constexpr uint32_t kCarry = 0x1FFFFF, kTop = 8;  // largest value 1.75 * 2^8
};
constexpr uint32_t kLeastScale = 16, kNoNumber = 255;

// One head's chunk of a page, in bytes.
template <int FMT, int D>
struct Chunk {
  static constexpr int kCode = D * Format<FMT>::kBits / 8;  // codes of one token
  static constexpr int kGroups = D / 32;
  static __device__ __host__ constexpr int64_t bytes(int block_size) {
    return int64_t(block_size) * (kCode + kGroups);
  }
};

struct QuantPages {
  const char* k;
  const char* v;
  int64_t page_bytes;
};

// Rows of values [token][head][D] with strides in elements; whole_words: every
// run of 16 bytes in a row is aligned.
struct Values {
  char* base;
  int64_t token, head;
  bool whole_words;
};

__device__ __forceinline__ const Header& header(const char* plan) {
  return *reinterpret_cast<const Header*>(plan);
}

// ------------------------------------------------------------ write, read --

struct SpanArgs {
  const char* plan;
  int64_t at_seqs, at_table;
  char* pages[2];       // K, V
  Values values[2];
  int64_t page_bytes;
  int32_t kv_heads, block_size;
  int32_t heads_each;   // heads one workgroup takes
  bool fresh;           // the new tokens, else all
};

// A span: up to 16 consecutive tokens of a sequence inside one block.
struct Span {
  int32_t block, inside, count;
  int64_t token;        // row of its first token among the values
};

__device__ __forceinline__ bool find_span(const SpanArgs& a, int32_t i, Span* s) {
  const Header& h = header(a.plan);
  if (i >= (a.fresh ? h.new_spans : h.read_spans)) return false;
  const Seq* seq = reinterpret_cast<const Seq*>(a.plan + a.at_seqs);
  // the last sequence that begins at or before span i; sequences without
  // spans begin where the next one does
  int32_t lo = 0, hi = h.num_seqs - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) >> 1;
    if ((a.fresh ? seq[mid].new_span : seq[mid].read_span) <= i) lo = mid;
    else hi = mid - 1;
  }
  const Seq q = seq[lo];
  const int32_t from = a.fresh ? q.len - q.fresh : 0;
  const int32_t nth = i - (a.fresh ? q.new_span : q.read_span);
  const int32_t grid = (from / kSpan + nth) * kSpan;
  const int32_t begin = max(grid, from), end = min(grid + kSpan, q.len);
  const int32_t column = begin / a.block_size;
  s->block = reinterpret_cast<const int32_t*>(a.plan + a.at_table)[q.table + column];
  s->inside = begin - column * a.block_size;
  s->count = end - begin;
  s->token = (a.fresh ? int64_t(q.token) : q.read_token) + (begin - from);
  return true;
}

// Eight values as float32, from 16-byte loads or one by one.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool whole_words, float* x) {
  T t[8];
  if (whole_words) {
    v4u w[sizeof(T) / 2];
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) w[i] = ((const gv4u*)p)[i];
    __builtin_memcpy(t, w, sizeof t);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(t[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool whole_words, const float* x) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = static_cast<T>(x[i]);
  if (whole_words) {
    v4u w[sizeof(T) / 2];
    __builtin_memcpy(w, t, sizeof t);
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) ((gv4u*)p)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = t[i];
  }
}

// The scale byte of a group whose largest magnitude has the bits `most`: the
// least e with most <= largest * 2^e, since adding kCarry carries into the
// exponent exactly where the mantissa is over the format's largest one.
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t most) {
  if (most >= 0x7F800000u) return kNoNumber;
  const int32_t b = static_cast<int32_t>((most + Format<FMT>::kCarry) >> 23) -
                    static_cast<int32_t>(Format<FMT>::kTop);
  return static_cast<uint32_t>(max(b, static_cast<int32_t>(kLeastScale)));
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

constexpr int kSpanLanes = 256;

// Write: eight values per lane, four lanes a group of 32. The scale is a power
// of two, so value / scale is exact and the hardware's rounding to nearest
// even is the only one.
template <int FMT, int D, typename T>
__global__ __launch_bounds__(kSpanLanes) void quant_write_kernel(SpanArgs a) {
  using C = Chunk<FMT, D>;
  constexpr int kLanesPerRow = D / 8;
  Span s;
  if (!find_span(a, blockIdx.x, &s)) return;
  const int kv = blockIdx.z;
  const int32_t head0 = blockIdx.y * a.heads_each;
  const int32_t heads = min(a.heads_each, a.kv_heads - head0);
  const Values& val = a.values[kv];
  const int64_t chunk = C::bytes(a.block_size);
  char* page = a.pages[kv] + s.block * a.page_bytes;
  const int part = threadIdx.x % kLanesPerRow;
  for (int32_t r = threadIdx.x / kLanesPerRow; r < heads * s.count;
       r += kSpanLanes / kLanesPerRow) {
    const int32_t h = r / s.count, t = r - h * s.count;
    float x[8];
    load8(reinterpret_cast<const T*>(val.base) + (s.token + t) * val.token +
              (head0 + h) * val.head + part * 8, val.whole_words, x);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 2)));
    const uint32_t byte = scale_byte<FMT>(most);
    const float scale = scale_of(byte);
    char* to = page + (head0 + h) * chunk;
    const int32_t at = s.inside + t;
    if constexpr (Format<FMT>::kBits == 4) {
      uint32_t c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
      if (byte == kNoNumber) c = 0;
      *reinterpret_cast<uint32_t*>(to + int64_t(at) * C::kCode + part * 4) = c;
    } else {
      s16x2 lo = {0, 0}, hi = {0, 0};
      lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[0], x[1], scale, false);
      lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[2], x[3], scale, true);
      hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[4], x[5], scale, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[6], x[7], scale, true);
      v2u c = {__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
      if (byte == kNoNumber) c = v2u{0, 0};
      *reinterpret_cast<v2u*>(to + int64_t(at) * C::kCode + part * 8) = c;
    }
    if (part % 4 == 0)
      to[int64_t(a.block_size) * C::kCode + (part / 4) * a.block_size + at] =
          static_cast<char>(byte);
  }
}

// The eight values of a lane's codes.
template <int FMT>
__device__ __forceinline__ void decode8(const uint32_t* c, float scale, float* x) {
  f32x2 p[4];
  if constexpr (Format<FMT>::kBits == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], scale, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[0], scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[0], scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[1], scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[1], scale, true);
  }
  __builtin_memcpy(x, p, 32);
}

template <int FMT, int D, typename T>
__global__ __launch_bounds__(kSpanLanes) void quant_read_kernel(SpanArgs a) {
  using C = Chunk<FMT, D>;
  constexpr int kLanesPerRow = D / 8;
  constexpr int kWords = Format<FMT>::kBits / 4;
  Span s;
  if (!find_span(a, blockIdx.x, &s)) return;
  const int kv = blockIdx.z;
  const int32_t head0 = blockIdx.y * a.heads_each;
  const int32_t heads = min(a.heads_each, a.kv_heads - head0);
  const Values& val = a.values[kv];
  const int64_t chunk = C::bytes(a.block_size);
  const char* page = a.pages[kv] + s.block * a.page_bytes;
  const int part = threadIdx.x % kLanesPerRow;
  for (int32_t r = threadIdx.x / kLanesPerRow; r < heads * s.count;
       r += kSpanLanes / kLanesPerRow) {
    const int32_t h = r / s.count, t = r - h * s.count;
    const char* from = page + (head0 + h) * chunk;
    const int32_t at = s.inside + t;
    uint32_t c[kWords];
    __builtin_memcpy(c, __builtin_assume_aligned(from + int64_t(at) * C::kCode + part * kWords * 4,
                                                 kWords * 4), kWords * 4);
    const uint32_t byte = static_cast<uint8_t>(
        from[int64_t(a.block_size) * C::kCode + (part / 4) * a.block_size + at]);
    float x[8];
    decode8<FMT>(c, scale_of(byte), x);
    if (byte == kNoNumber) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(0x7FC00000u);
    }
    store8(reinterpret_cast<T*>(val.base) + (s.token + t) * val.token +
               (head0 + h) * val.head + part * 8, val.whole_words, x);
  }
}

// --------------------------------------------------------------- attention --

// Matrix operands in the queries' type. The cache's values are exact in
// bfloat16 and, between 2^-24 and its largest value, in float16.
template <typename T>
struct Operand;
template <>
struct Operand<__bf16> {
  typedef bf16x8 v8;
  // probabilities lie in [0, 2^kLift]
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t fp4(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t fp8(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, SEL != 0));
  }
};
template <>
struct Operand<_Float16> {
  typedef f16x8 v8;
  // float16 keeps 2^-24 at the least: lifted, small probabilities of long
  // contexts are not lost beside the largest one (the sum is lifted alike)
  static constexpr float kLift = 14.f;
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t fp4(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, SEL));
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t fp8(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, SEL != 0));
  }
};

// Pair PAIR (values 2 PAIR, 2 PAIR + 1) of a lane's code words, as two values.
template <int FMT, typename T, int PAIR>
__device__ __forceinline__ uint32_t decode_pair(const uint32_t* w, float s) {
  if constexpr (Format<FMT>::kBits == 4)
    return Operand<T>::template fp4<PAIR % 4>(w[PAIR / 4], s);
  else
    return Operand<T>::template fp8<PAIR % 2>(w[PAIR / 2], s);
}

struct AttendArgs {
  const char* plan;
  int64_t at_seqs, at_table, at_items, at_merges;
  QuantPages pages;
  Values q, out;
  float* work;          // parts of this kind's items, by slot
  int64_t slot_floats;
  int64_t kind_work[kKinds];   // merge: where each kind's parts begin
  float* work_base;
  int64_t kind_slot_floats[kKinds];
  float c;              // scale * log2(e)
  int32_t block_shift, group, window, sinks;
  int32_t kind;
};

// A wave's tile of 32 tokens as it lies in the cache. Lane l (m = l % 16, g = l
// / 16) holds of K, for both halves of 16 tokens, token m's values [D/4 g, D/4 (g
// + 1)), and of V the values [D/16 m, D/16 (m + 1)) of tokens 4g .. 4g + 3 of
// each half: what its matrix operands are made of, without any exchange. The
// order of the tokens and values along a product's inner axis is free, so it
// is the one in which they were loaded.
template <int FMT, int D>
struct CacheTile {
  static constexpr int kKWords = Chunk<FMT, D>::kCode / 16;
  static constexpr int kVBytes = Chunk<FMT, D>::kCode / 16;
  static constexpr int kVWords = (kVBytes + 3) / 4;
  static constexpr int kKScales = D == 256 ? 2 : 1;
  uint32_t k[2][kKWords];
  uint32_t ks[2][kKScales];
  uint32_t v[2][4][kVWords];
  uint32_t vs[2];       // four tokens' scale bytes

  __device__ __forceinline__ void load(const QuantPages& p, int64_t head_offset,
                                       int block_shift, const int32_t* table, int32_t tile, int m,
                                       int g) {
    using C = Chunk<FMT, D>;
    const int32_t block_size = 1 << block_shift;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int32_t position = tile * kTile + half * 16;
      const int32_t column = position >> block_shift;
      const int32_t inside = position - (column << block_shift);
      const int64_t at = int64_t(table[column]) * p.page_bytes + head_offset;
      const char* kc = p.k + at + inside * C::kCode;
      const char* vc = p.v + at + inside * C::kCode;
      const char* ksc = p.k + at + block_size * C::kCode + inside;
      const char* vsc = p.v + at + block_size * C::kCode + inside;
      constexpr int kKBytes = kKWords * 4;
      __builtin_memcpy(k[half],
                       __builtin_assume_aligned(kc + m * C::kCode + g * kKBytes,
                                                kKBytes < 16 ? kKBytes : 16), kKBytes);
#pragma unroll
      for (int i = 0; i < kKScales; ++i)
        ks[half][i] = static_cast<uint8_t>(
            ksc[(D == 64 ? g / 2 : g * kKScales + i) * block_size + m]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* t = vc + (4 * g + i) * C::kCode + m * kVBytes;
        if constexpr (kVBytes == 2) {
          v[half][i][0] = *reinterpret_cast<const uint16_t*>(t);
        } else {
          __builtin_memcpy(v[half][i], __builtin_assume_aligned(t, kVBytes), kVBytes);
        }
      }
      vs[half] = *reinterpret_cast<const uint32_t*>(vsc + (m * D / 512) * block_size + 4 * g);
    }
  }
};

// largest of a value over the four lanes of a row (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float row_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float row_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// f(0), .., f(N - 1) with constants
template <int I, int N, typename F>
__device__ __forceinline__ void each_constant(const F& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each_constant<I + 1, N>(f);
  }
}

// Whether a query at position p sees position j (window: INT32_MAX for none).
__device__ __forceinline__ bool seen(const AttendArgs& a, int32_t p, int32_t j) {
  return (j <= p) & ((p - j < a.window) | (j < a.sinks));
}

constexpr int kAttendLanes = 256, kAttendWaves = 4;

template <int FMT, int D, typename T, int R>
__global__ __launch_bounds__(kAttendLanes) void quant_attend_kernel(AttendArgs a) {
  typedef typename Operand<T>::v8 v8;
  using Tile = CacheTile<FMT, D>;
  constexpr int kSteps = D / 32;    // matrix steps along the head
  constexpr int kOut = D / 16;      // output tiles of 16 values
  constexpr int kPad = D + 4;
  __shared__ float joined[kAttendWaves][16][kPad];
  __shared__ float stats[2][kAttendWaves][16 * R];

  const Header& h = header(a.plan);
  if (static_cast<int32_t>(blockIdx.x) >= h.items[a.kind]) return;
  const Item it = reinterpret_cast<const Item*>(a.plan + a.at_items)[blockIdx.x];
  const Seq seq = reinterpret_cast<const Seq*>(a.plan + a.at_seqs)[it.seq];
  const int32_t* table = reinterpret_cast<const int32_t*>(a.plan + a.at_table) + seq.table;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, m = lane % 16, g = lane / 16;
  const int64_t head_offset = it.kv_head * Chunk<FMT, D>::bytes(1 << a.block_shift);

  // queries: row m of each row tile, its values [D/4 g, D/4 (g + 1))
  v8 q[R][kSteps];
  int32_t position[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int32_t row = it.row + 16 * r + m;
    const bool there = 16 * r + m < it.rows;
    const int32_t token = row / a.group;
    position[r] = seq.len - seq.fresh + (there ? token : 0);
    const T* from = reinterpret_cast<const T*>(a.q.base) + (int64_t(seq.token) + token) * a.q.token +
                    (int64_t(it.kv_head) * a.group + (row - token * a.group)) * a.q.head + g * (D / 4);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int j = 0; j < 8; ++j) q[r][s][j] = there ? from[s * 8 + j] : T(0.f);
    }
  }
  const int32_t base = seq.len - seq.fresh;
  const int32_t low = base + it.row / a.group, high = base + (it.row + it.rows - 1) / a.group;

  f32x4 o[R][kOut];
  float top[R], sum[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    top[r] = -INFINITY;
    sum[r] = 0.f;
#pragma unroll
    for (int d = 0; d < kOut; ++d) o[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto tile_at = [&](int32_t v) {
    return v < it.first_tiles ? v : v - it.first_tiles + it.window_tile;
  };
  Tile cur;
  int32_t at = it.tile + wave;
  if (at < it.tile_end)
    cur.load(a.pages, head_offset, a.block_shift, table, tile_at(at), m, g);
  for (; at < it.tile_end; at += kAttendWaves) {
    const int32_t tile = tile_at(at);
    Tile next = cur;
    if (at + kAttendWaves < it.tile_end)
      next.load(a.pages, head_offset, a.block_shift, table, tile_at(at + kAttendWaves), m, g);

    // scores: lane holds row m, tokens 4g + i of both halves
    f32x4 x[R][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const float scale = scale_of(cur.ks[half][Tile::kKScales == 2 ? s / 4 : 0]);
        const uint32_t* w = &cur.k[half][s * Format<FMT>::kBits / 4];
        uint32_t f[4];
        f[0] = decode_pair<FMT, T, 0>(w, scale);
        f[1] = decode_pair<FMT, T, 1>(w, scale);
        f[2] = decode_pair<FMT, T, 2>(w, scale);
        f[3] = decode_pair<FMT, T, 3>(w, scale);
        v8 kf;
        __builtin_memcpy(&kf, f, 16);
#pragma unroll
        for (int r = 0; r < R; ++r) x[r][half] = Operand<T>::mma(kf, q[r][s], x[r][half]);
      }
    }

    // Tokens that some row does not see; in other tiles every row sees every
    // token. All by selection: with branches around the changed elements the
    // compiler lost one of the changes (the first element's, its operands being
    // copied out of the matrix registers in several places).
    const int32_t begin = tile * kTile;
    const bool whole = (begin + kTile - 1 <= low) &
                       ((high - begin < a.window) | (begin + kTile <= a.sinks));
    uint32_t odd = 0;   // seen tokens (bit 4 half + i) whose V is no number
    if (!whole) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t j = begin + 16 * half + 4 * g + i;
#pragma unroll
          for (int r = 0; r < R; ++r)
            x[r][half][i] = seen(a, position[r], j) ? x[r][half][i] : -INFINITY;
          // what no row sees may hold anything: its product with a
          // probability of 0 has to be 0
          const bool any = (j <= high) & ((low - j < a.window) | (j < a.sinks));
          const uint32_t byte = (cur.vs[half] >> (8 * i)) & 255u;
          const bool number = byte != kNoNumber;
          odd |= any & !number ? 1u << (4 * half + i) : 0u;
          const uint32_t keep = any & number ? ~0u : 0u;
          cur.vs[half] = (cur.vs[half] & ~(255u << (8 * i))) | ((keep ? byte : 127u) << (8 * i));
#pragma unroll
          for (int w = 0; w < Tile::kVWords; ++w) cur.v[half][i][w] &= keep;
        }
      }
    }

    v8 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float most = fmaxf(fmaxf(fmaxf(x[r][0][0], x[r][0][1]), fmaxf(x[r][0][2], x[r][0][3])),
                         fmaxf(fmaxf(x[r][1][0], x[r][1][1]), fmaxf(x[r][1][2], x[r][1][3])));
      most = fmaxf(top[r], row_max(most));
      if (__any(most > top[r])) {
        const float fade = top[r] == most ? 1.f : __builtin_amdgcn_exp2f((top[r] - most) * a.c);
        sum[r] *= fade;
#pragma unroll
        for (int d = 0; d < kOut; ++d) o[r][d] *= fade;
        top[r] = most;
      }
      const float lift = Operand<T>::kLift - (most == -INFINITY ? 0.f : most * a.c);
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r][i / 4][i % 4], a.c, lift));
        sum[r] += e[i];
        p[r][i] = static_cast<T>(e[i]);
      }
    }

    // values: pairs of tokens side by side, one operand per value of the lane
    float vscale[2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < 4; ++i) vscale[half][i] = scale_of((cur.vs[half] >> (8 * i)) & 255u);
    auto values = [&](auto pair) {
      constexpr int B = decltype(pair)::value;
      uint32_t even[4], oddv[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int half = t / 2, i = 2 * (t % 2);
        const uint32_t c0 = decode_pair<FMT, T, B>(cur.v[half][i], vscale[half][i]);
        const uint32_t c1 = decode_pair<FMT, T, B>(cur.v[half][i + 1], vscale[half][i + 1]);
        even[t] = __builtin_amdgcn_perm(c1, c0, 0x05040100u);
        oddv[t] = __builtin_amdgcn_perm(c1, c0, 0x07060302u);
      }
      v8 f0, f1;
      __builtin_memcpy(&f0, even, 16);
      __builtin_memcpy(&f1, oddv, 16);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        o[r][2 * B] = Operand<T>::mma(f0, p[r], o[r][2 * B]);
        o[r][2 * B + 1] = Operand<T>::mma(f1, p[r], o[r][2 * B + 1]);
      }
    };
    each_constant<0, kOut / 2>(values);

    // Rows that see a V that is no number are none there; the others, in whose
    // product it had to count as 0, stay as they are. Lane l of the operand
    // knows the groups of values [D/16 m, ..), of the result [D/4 g, ..).
    if (__any(odd != 0)) {
      for (int t = 0; t < kTile; ++t) {
        const int owner_g = (t % 16) / 4, bit = 4 * (t / 16) + t % 4;
        const int32_t j = begin + t;
#pragma unroll
        for (int grp = 0; grp < D / 32; ++grp) {
          // a lane of the operand that holds this token and group
          const int from = owner_g * 16 + grp * 512 / D;
          const bool none = (__shfl(static_cast<int>(odd), from) >> bit) & 1;
          if (!none) continue;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const bool sees = seen(a, position[r], j);
#pragma unroll
            for (int d = 0; d < kOut; ++d)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int value = (D / 16) * (4 * g + i) + d;
                o[r][d][i] = sees & (value / 32 == grp) ? __uint_as_float(0x7FC00000u)
                                                        : o[r][d][i];
              }
          }
        }
      }
    }
    cur = next;
  }

  // join the waves: each scales its part to the largest score of all
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float s = row_sum(sum[r]);
    if (g == 0) {
      stats[0][wave][16 * r + m] = top[r];
      stats[1][wave][16 * r + m] = s;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float most = stats[0][0][16 * r + m];
#pragma unroll
    for (int w = 1; w < kAttendWaves; ++w) most = fmaxf(most, stats[0][w][16 * r + m]);
    const float fade = top[r] == most ? 1.f : __builtin_amdgcn_exp2f((top[r] - most) * a.c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kOut; ++d)
        joined[wave][m][(D / 16) * (4 * g + i) + d] = o[r][d][i] * fade;
    __syncthreads();
    const int row = threadIdx.x / 16, part = threadIdx.x % 16;
    if (16 * r + row < it.rows) {
      float all = stats[0][0][16 * r + row], total = 0.f;
#pragma unroll
      for (int w = 1; w < kAttendWaves; ++w) all = fmaxf(all, stats[0][w][16 * r + row]);
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        const float t = stats[0][w][16 * r + row];
        total += stats[1][w][16 * r + row] * (t == all ? 1.f : __builtin_amdgcn_exp2f((t - all) * a.c));
      }
      float y[D / 16];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        y[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w) y[i] += joined[w][row][part * (D / 16) + i];
      }
      if (it.slot < 0) {
        const int32_t n = it.row + 16 * r + row, token = n / a.group;
        T* to = reinterpret_cast<T*>(a.out.base) + (int64_t(seq.token) + token) * a.out.token +
                (int64_t(it.kv_head) * a.group + (n - token * a.group)) * a.out.head;
        const float inv = 1.f / total;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) to[part * (D / 16) + i] = static_cast<T>(y[i] * inv);
      } else {
        float* to = a.work + it.slot * a.slot_floats + (16 * r + row) * (D + 2);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) to[part * (D / 16) + i] = y[i];
        if (part == 0) {
          to[D] = all;
          to[D + 1] = total;
        }
      }
    }
    __syncthreads();
  }
}

// Rows whose tiles several items shared: one workgroup a row, 256 / D parts
// side by side.
template <int D, typename T>
__global__ __launch_bounds__(256) void quant_merge_kernel(AttendArgs a) {
  constexpr int kSide = 256 / D;
  __shared__ float side[kSide][D];
  __shared__ float side_sum[kSide];
  const Header& h = header(a.plan);
  if (static_cast<int32_t>(blockIdx.x) >= h.merges) return;
  const Merge mg = reinterpret_cast<const Merge*>(a.plan + a.at_merges)[blockIdx.x];
  const int row = blockIdx.y;
  if (row >= mg.rows) return;
  const Seq seq = reinterpret_cast<const Seq*>(a.plan + a.at_seqs)[mg.seq];
  const int64_t each = a.kind_slot_floats[mg.kind];
  const float* from = a.work_base + a.kind_work[mg.kind] + mg.slot * each + row * (D + 2);
  float most = -INFINITY;
  for (int p = 0; p < mg.parts; ++p) most = fmaxf(most, from[p * each + D]);
  const int d = threadIdx.x % D, s = threadIdx.x / D;
  float y = 0.f, total = 0.f;
  for (int p = s; p < mg.parts; p += kSide) {
    const float t = from[p * each + D];
    const float fade = t == most ? 1.f : __builtin_amdgcn_exp2f((t - most) * a.c);
    y += fade * from[p * each + d];
    total += fade * from[p * each + D + 1];
  }
  side[s][d] = y;
  if (d == 0) side_sum[s] = total;
  __syncthreads();
  if (s != 0) return;
#pragma unroll
  for (int i = 1; i < kSide; ++i) {
    y += side[i][d];
    total += side_sum[i];
  }
  const int32_t n = mg.row + row, token = n / a.group;
  T* to = reinterpret_cast<T*>(a.out.base) + (int64_t(seq.token) + token) * a.out.token +
          (int64_t(mg.kv_head) * a.group + (n - token * a.group)) * a.out.head;
  to[d] = static_cast<T>(y / total);
}

}  // namespace

#endif  // AEGKV_QUANT_CACHE_H
