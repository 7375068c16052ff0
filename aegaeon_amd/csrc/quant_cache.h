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

// The plan does not change while a kernel runs. Read as constant memory, what is
// the same for a wave comes by scalar loads; as ordinary memory, once a kernel
// stores anything, by vector loads in one queue with the cache's, and waiting
// for a block id meant waiting for every tile on its way.
#define AEGKV_CONSTANT __attribute__((address_space(4)))

template <typename T>
__device__ __forceinline__ const AEGKV_CONSTANT T* in_plan(const char* plan, int64_t offset) {
  return (const AEGKV_CONSTANT T*)(reinterpret_cast<uintptr_t>(plan) +
                                   static_cast<uintptr_t>(offset));
}

// The same address, to read from anew: what few steps need is not held in scalar
// registers (a hundred, and spilled ones cost vector instructions) in between.
template <typename P>
__device__ __forceinline__ P anew(P p) {
  asm volatile("" : "+s"(p));
  return p;
}

// ------------------------------------------------------------ write, read --

struct SpanArgs {
  const char* plan;
  int64_t at_seqs, at_table, at_new_spans;
  char* pages[2];       // K, V
  Values values[2];
  int64_t page_bytes;
  int32_t kv_heads, block_size;
  // Workgroup i takes heads_each heads of span i / head_groups: neighbours work
  // on neighbouring memory (with the spans first, prompts were written in 92 us, not 85).
  int32_t heads_each, head_groups;
  bool fresh;           // the new tokens, else all
};

// A span: up to 16 consecutive tokens of a sequence inside one block.
struct Span {
  int32_t block, inside, count;
  int64_t token;        // row of its first token among the values
};

__device__ __forceinline__ bool find_span(const SpanArgs& a, int32_t i, Span* s) {
  const auto* h = in_plan<Header>(a.plan, 0);
  if (a.fresh) {
    const auto* n = in_plan<NewSpan>(a.plan, a.at_new_spans) + i;
    *s = Span{n->block, n->inside, n->count, n->token};
    return i < h->new_spans;
  }
  // a captured read may find, after an update, a batch with released columns
  if (i >= h->read_spans || !h->complete) return false;
  const auto* seq = in_plan<Seq>(a.plan, a.at_seqs);
  // the last sequence that begins at or before span i; empty sequences begin
  // where the next one does
  int32_t lo = 0, hi = h->num_seqs - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) >> 1;
    if (seq[mid].read_span <= i) lo = mid;
    else hi = mid - 1;
  }
  const auto* q = seq + lo;
  const int32_t begin = (i - q->read_span) * kSpan;
  const int32_t column = begin / a.block_size;
  s->block = in_plan<int32_t>(a.plan, a.at_table)[q->table + column];
  s->inside = begin - column * a.block_size;
  s->count = min(kSpan, q->len - begin);
  s->token = q->read_token + begin;
  return true;
}

// Eight values as float32, from 16-byte loads or one by one.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool whole_words, float* x) {
  T t[8];
  if (whole_words) {
    v4u w[sizeof(T) / 2];
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i)
      w[i] = __builtin_nontemporal_load((const gv4u*)p + i);
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
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) __builtin_nontemporal_store(w[i], (gv4u*)p + i);
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

// A group's codes as they are stored: a lane's eight values, four lanes a group.
// The scale is a power of two, so value / scale is exact and the hardware's
// rounding to nearest even is the only one.
template <int FMT>
struct Codes {
  static constexpr int kWords = Format<FMT>::kBits / 4;
  uint32_t w[kWords];
  uint32_t byte;        // the group's scale

  __device__ __forceinline__ void encode(const float* x) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 2)));
    byte = scale_byte<FMT>(most);
    const float scale = scale_of(byte);
    if constexpr (Format<FMT>::kBits == 4) {
      uint32_t c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
      w[0] = byte == kNoNumber ? 0 : c;
    } else {
      s16x2 lo = {0, 0}, hi = {0, 0};
      lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[0], x[1], scale, false);
      lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[2], x[3], scale, true);
      hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[4], x[5], scale, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[6], x[7], scale, true);
      w[0] = byte == kNoNumber ? 0 : __builtin_bit_cast(uint32_t, lo);
      w[1] = byte == kNoNumber ? 0 : __builtin_bit_cast(uint32_t, hi);
    }
  }

  __device__ __forceinline__ void decode(float* x) const {
    const float scale = scale_of(byte);
    f32x2 p[4];
    if constexpr (Format<FMT>::kBits == 4) {
      p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], scale, 0);
      p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], scale, 1);
      p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], scale, 2);
      p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], scale, 3);
    } else {
      p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[0], scale, false);
      p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[0], scale, true);
      p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[1], scale, false);
      p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[1], scale, true);
    }
    __builtin_memcpy(x, p, 32);
    if (byte == kNoNumber) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(0x7FC00000u);
    }
  }
};

// A workgroup's rows: `count` tokens of each of `heads` heads, D / 8 lanes a row.
// kAtOnce rows of a lane are on their way together.
constexpr int kAtOnce = 4;

template <int D>
struct SpanWalk {
  static constexpr int kRowLanes = D / 8, kRows = kSpanLanes / kRowLanes;
  Span s;
  int32_t head0, rows;
  int part, first;

  __device__ __forceinline__ bool begin(const SpanArgs& a) {
    const int32_t span = blockIdx.x / a.head_groups;
    if (!find_span(a, span, &s)) return false;
    head0 = (blockIdx.x - span * a.head_groups) * a.heads_each;
    rows = min(a.heads_each, a.kv_heads - head0) * s.count;
    part = threadIdx.x % kRowLanes;
    first = threadIdx.x / kRowLanes;
    return true;
  }
  // (head, token) of row r
  __device__ __forceinline__ void find(int32_t r, int32_t* h, int32_t* t) const {
    if (s.count == kSpan) {
      *h = r / kSpan;
      *t = r % kSpan;
    } else {
      *h = r / s.count;
      *t = r - *h * s.count;
    }
  }
};

// Write: e = least power with max |x| <= largest * 2^e over a group of 32, codes
// rne(x 2^-e). Bound by HBM: 12,300 prompt tokens of 40 heads, 128 wide, bfloat16
// to mxfp4 (251 MB read, 66 written) take 62 us, 5.1 TB/s. Values come past the
// caches (85 us when they went through), the heads of a span are neighbouring
// workgroups; codes and scales stay in the L2, where attention looks for them next.
template <int FMT, int D, typename T>
__global__ __launch_bounds__(kSpanLanes) void quant_write_kernel(SpanArgs a) {
  using C = Chunk<FMT, D>;
  using Walk = SpanWalk<D>;
  constexpr int kWords = Codes<FMT>::kWords;
  Walk walk;
  if (!walk.begin(a)) return;
  const Span& s = walk.s;
  const Values val = a.values[blockIdx.y];
  const int64_t chunk = C::bytes(a.block_size);
  char* page = a.pages[blockIdx.y] + s.block * a.page_bytes + walk.head0 * chunk;
  const T* from = reinterpret_cast<const T*>(val.base) + s.token * val.token +
                  walk.head0 * val.head + walk.part * 8;
  for (int32_t r0 = walk.first; r0 < walk.rows; r0 += Walk::kRows * kAtOnce) {
    float x[kAtOnce][8];
    int32_t h[kAtOnce], t[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      // rows behind the last one are read again, not past it
      walk.find(min(r0 + u * Walk::kRows, walk.rows - 1), &h[u], &t[u]);
      load8(from + t[u] * val.token + h[u] * val.head, val.whole_words, x[u]);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      Codes<FMT> c;
      c.encode(x[u]);
      if (r0 + u * Walk::kRows >= walk.rows) continue;
      char* to = page + h[u] * chunk;
      const int32_t at = s.inside + t[u];
      __builtin_memcpy(__builtin_assume_aligned(to + at * C::kCode + walk.part * kWords * 4,
                                                kWords * 4), c.w, kWords * 4);
      if (walk.part % 4 == 0)
        to[a.block_size * C::kCode + (walk.part / 4) * a.block_size + at] =
            static_cast<char>(c.byte);
    }
  }
}

// Read: x = code * 2^(byte - 127), rounded once. Bound by HBM: the same tokens
// back take 50 us (6.3 TB/s), 24 contexts of 8 heads (552 MB) 99 us (5.6 TB/s).
template <int FMT, int D, typename T>
__global__ __launch_bounds__(kSpanLanes) void quant_read_kernel(SpanArgs a) {
  using C = Chunk<FMT, D>;
  using Walk = SpanWalk<D>;
  constexpr int kWords = Codes<FMT>::kWords;
  Walk walk;
  if (!walk.begin(a)) return;
  const Span& s = walk.s;
  const Values val = a.values[blockIdx.y];
  const int64_t chunk = C::bytes(a.block_size);
  const char* page = a.pages[blockIdx.y] + s.block * a.page_bytes + walk.head0 * chunk;
  T* to = reinterpret_cast<T*>(val.base) + s.token * val.token + walk.head0 * val.head +
          walk.part * 8;
  for (int32_t r0 = walk.first; r0 < walk.rows; r0 += Walk::kRows * kAtOnce) {
    Codes<FMT> c[kAtOnce];
    int32_t h[kAtOnce], t[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      walk.find(min(r0 + u * Walk::kRows, walk.rows - 1), &h[u], &t[u]);
      const char* from = page + h[u] * chunk;
      const int32_t at = s.inside + t[u];
      __builtin_memcpy(c[u].w,
                       __builtin_assume_aligned(from + at * C::kCode + walk.part * kWords * 4,
                                                kWords * 4), kWords * 4);
      c[u].byte = static_cast<uint8_t>(
          from[a.block_size * C::kCode + (walk.part / 4) * a.block_size + at]);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (r0 + u * Walk::kRows >= walk.rows) continue;
      float x[8];
      c[u].decode(x);
      store8(to + t[u] * val.token + h[u] * val.head, val.whole_words, x);
    }
  }
}

// --------------------------------------------------------------- attention --

// Matrix operands in the queries' type. The cache's values are exact in
// bfloat16 and, between 2^-24 and its largest value, in float16. Groups whose scale
// byte is kFar or more may hold values beyond that (4 or 256 times the scale), or no
// number.
template <typename T>
struct Operand;
template <>
struct Operand<__bf16> {
  typedef bf16x8 v8;
  static constexpr float kLift = 0.f, kLimit = 65536.f;
  template <int FMT>
  static constexpr uint32_t kFar = Format<FMT>::kBits == 4 ? 253 : 247;   // 2^128
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
  // float16 keeps 2^-24 at the least and 2^16 at the most: lifted, small
  // probabilities of long contexts are not lost beside the largest one (the sum
  // is lifted alike), and a row may still grow 2^8-fold
  static constexpr float kLift = 7.f, kLimit = 32768.f;
  template <int FMT>
  static constexpr uint32_t kFar = Format<FMT>::kBits == 4 ? 141 : 135;   // 2^16
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

// What every step of attention needs.
struct Scope {
  QuantPages pages;
  float c;              // scale * log2(e)
  int32_t block_shift, window, sinks;
};

struct AttendArgs {
  Scope scope;
  const char* plan;
  int64_t at_table, at_items, at_merges;
  Values q, out;
  float* work;          // parts of this kind's items, by slot
  int64_t slot_floats;
  int64_t kind_work[kKinds];   // merge: where each kind's parts begin
  float* work_base;
  int64_t kind_slot_floats[kKinds];
  int32_t group, kind;
};

typedef const AEGKV_CONSTANT AttendArgs* ColdArgs;
typedef const AEGKV_CONSTANT Item* ItemPtr;

// A kernel's only argument, read where it is needed.
__device__ __forceinline__ ColdArgs cold_args() {
  return anew((ColdArgs)__builtin_amdgcn_kernarg_segment_ptr());
}

// A wave's tile of 32 tokens as it lies in the cache. Lane l (m = l % 16, g = l
// / 16) holds of K, for both halves of 16 tokens, token m's values [D/4 g, D/4 (g
// + 1)), and of V the values [D/16 m, D/16 (m + 1)) of tokens 4g .. 4g + 3 of
// each half: what its matrix operands are made of, without any exchange. The
// order of the tokens and values along a product's inner axis is free, so it
// is the one in which they were loaded.

// Where a half of 16 tokens lies: the same for the whole wave, so that a load is
// a scalar address and a lane's own 32-bit offset.
struct Half {
  const char* k;        // codes of its first token
  const char* v;
  const char* k_scales;
  const char* v_scales;
};

template <int FMT, int D>
__device__ __forceinline__ Half find_half(const QuantPages& p, int64_t head_offset,
                                          int block_shift, int32_t block, int32_t position) {
  using C = Chunk<FMT, D>;
  const int32_t inside = position & ((1 << block_shift) - 1);
  const int64_t at = int64_t(block) * p.page_bytes + head_offset;
  const int64_t codes = at + int64_t(inside) * C::kCode;
  const int64_t scales = at + (int64_t(C::kCode) << block_shift) + inside;
  return Half{p.k + codes, p.v + codes, p.k + scales, p.v + scales};
}

// STREAM: past the caches, for what mostly one workgroup reads (64 decodes of one
// token 58 us, through them 62). Second readers find less: the two blocks of 33 to 64
// rows of a sequence (40 rows 69 us, through them 67; 64 rows 70 both ways) and sequences
// that share blocks (64 decodes over a common 4,000 tokens 46 us, through them 43.5).
template <int BYTES, bool STREAM>
__device__ __forceinline__ void load_bytes(uint32_t* to, const char* base, uint32_t offset) {
  const char* p = base + offset;
  const auto one = [](const auto* at) {
    return STREAM ? __builtin_nontemporal_load(at) : *at;
  };
  if constexpr (BYTES == 1) {
    to[0] = one(reinterpret_cast<const uint8_t*>(p));
  } else if constexpr (BYTES == 2) {
    to[0] = one(reinterpret_cast<const uint16_t*>(p));
  } else if constexpr (BYTES == 4) {
    to[0] = one(reinterpret_cast<const uint32_t*>(p));
  } else if constexpr (BYTES == 8) {
    const v2u x = one(reinterpret_cast<const v2u*>(p));
    __builtin_memcpy(to, &x, 8);
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const v4u x = one(reinterpret_cast<const v4u*>(p) + i);
      __builtin_memcpy(to + 4 * i, &x, 16);
    }
  }
}

// A lane's part of 16 tokens of K, and the scales of its groups.
template <int FMT, int D, bool STREAM>
struct KPart {
  static constexpr int kWords = Chunk<FMT, D>::kCode / 16;
  static constexpr int kScales = D == 256 ? 2 : 1;
  uint32_t code[kWords], scale[kScales];

  __device__ __forceinline__ void load(const Half& h, int block_shift, uint32_t m, uint32_t g) {
    load_bytes<kWords * 4, STREAM>(code, h.k, m * Chunk<FMT, D>::kCode + g * (kWords * 4));
#pragma unroll
    for (uint32_t i = 0; i < kScales; ++i)
      load_bytes<1, STREAM>(&scale[i], h.k_scales,
                            ((D == 64 ? g / 2 : g * kScales + i) << block_shift) + m);
  }

  // The matrix operand of step S: the lane's values 8 S .. 8 S + 7.
  template <typename T, int S>
  __device__ __forceinline__ typename Operand<T>::v8 operand() const {
    const float s = scale_of(scale[kScales == 2 ? S / 4 : 0]);
    const uint32_t* w = &code[S * Format<FMT>::kBits / 4];
    const uint32_t f[4] = {decode_pair<FMT, T, 0>(w, s), decode_pair<FMT, T, 1>(w, s),
                           decode_pair<FMT, T, 2>(w, s), decode_pair<FMT, T, 3>(w, s)};
    typename Operand<T>::v8 k;
    __builtin_memcpy(&k, f, 16);
    return k;
  }
};

// A lane's part of 32 tokens of V: BYTES of each of its eight tokens, from byte
// `from` of the lane's on.
template <int FMT, int D, int BYTES, bool STREAM>
struct VPart {
  static constexpr int kWords = (BYTES + 3) / 4;
  static constexpr int kPairs = BYTES * 4 / Format<FMT>::kBits;   // pairs of values
  uint32_t code[2][4][kWords], scale[2];    // scale: a byte for each of four tokens

  __device__ __forceinline__ void load(const Half* h, int block_shift, uint32_t m, uint32_t g,
                                       uint32_t from) {
    constexpr uint32_t kCode = Chunk<FMT, D>::kCode;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        load_bytes<BYTES, STREAM>(code[half][i], h[half].v + i * kCode,
                          4 * g * kCode + m * (kCode / 16) + from);
      load_bytes<4, STREAM>(&scale[half], h[half].v_scales, ((m * D / 512) << block_shift) + 4 * g);
    }
  }

  // Whether a group may hold what is no operand of the queries' type: some scale
  // byte reaches kFar (a byte's low bits carry into its top one, which is set).
  template <typename T>
  __device__ __forceinline__ bool far() const {
    constexpr uint32_t kFar = Operand<T>::template kFar<FMT>;
    static_assert(kFar >= 128, "the byte's top bit is set");
    uint32_t found = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half)
      found |= ((scale[half] & 0x7F7F7F7Fu) + (256 - kFar) * 0x01010101u) & scale[half];
    return (found & 0x80808080u) != 0;
  }

  // What no row of [low, high] sees may hold anything: its product with a
  // probability of 0 has to be 0. Returns the seen tokens (bit 4 half + i) whose
  // values here are no operands of the queries' type, or are no numbers; they count
  // as 0 too, for the rows that do not see them, and add_far adds them for the others.
  template <typename T>
  __device__ __forceinline__ uint32_t clear(int32_t begin, int32_t g, int32_t low, int32_t high,
                                            int32_t window, int32_t sinks) {
    uint32_t odd = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t j = begin + 16 * half + 4 * g + i;
        const bool any = (j <= high) & ((low - j < window) | (j < sinks));
        const uint32_t byte = (scale[half] >> (8 * i)) & 255u;
        bool number = byte < Operand<T>::template kFar<FMT>;
        if constexpr (Format<FMT>::kBits == 8) {   // E4M3 has codes that are none
#pragma unroll
          for (int w = 0; w < kWords; ++w)
            number &= (((code[half][i][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) == 0;
        }
        odd |= (any & !number) ? 1u << (4 * half + i) : 0u;
        const uint32_t keep = (any & number) ? ~0u : 0u;
        scale[half] = (scale[half] & ~(255u << (8 * i))) | ((keep ? byte : 127u) << (8 * i));
#pragma unroll
        for (int w = 0; w < kWords; ++w) code[half][i][w] &= keep;
      }
    }
    return odd;
  }

  __device__ __forceinline__ void scales(float (*s)[4]) const {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[half][i] = scale_of((scale[half] >> (8 * i)) & 255u);
  }

  // The operands of values 2 B and 2 B + 1: eight tokens side by side each.
  template <typename T, int B>
  __device__ __forceinline__ void operands(const float (*s)[4], typename Operand<T>::v8* even,
                                           typename Operand<T>::v8* odd) const {
    uint32_t e[4], o[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int half = t / 2, i = 2 * (t % 2);
      const uint32_t c0 = decode_pair<FMT, T, B>(code[half][i], s[half][i]);
      const uint32_t c1 = decode_pair<FMT, T, B>(code[half][i + 1], s[half][i + 1]);
      e[t] = __builtin_amdgcn_perm(c1, c0, 0x05040100u);
      o[t] = __builtin_amdgcn_perm(c1, c0, 0x07060302u);
    }
    __builtin_memcpy(even, e, 16);
    __builtin_memcpy(odd, o, 16);
  }
};

// largest of a value over the four lanes of a row (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float row_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
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
__device__ __forceinline__ bool seen(const Scope& a, int32_t p, int32_t j) {
  return (j <= p) & ((p - j < a.window) | (j < a.sinks));
}

// The tokens of `odd` (a lane's bits, as VPart::clear gives them): bit m for token t of the
// tile where lane m of its four tokens' has it.
__device__ __forceinline__ uint32_t lanes_of(uint32_t odd, int t) {
  const uint64_t all = __ballot((odd >> (4 * (t / 16) + t % 4)) & 1);
  return static_cast<uint32_t>(all >> (16 * (t % 16 / 4))) & 0xFFFFu;
}

// Adds to the rows of R row tiles that see them, in 32 bits, the tokens that
// were cleared from V's operands: values [FIRST, FIRST + COUNT) of the runs [D/16 m, D/16
// (m + 1)) with m in who(t), which is the same for the whole wave. Read anew from
// the cache, a token at a time: they are rare. By selection, as above where scores
// are hidden.
template <int FMT, int D, typename T, int R, int FIRST, int COUNT, typename W>
__device__ __forceinline__ void add_far(const Scope& a, const W& who,
                                        const AEGKV_CONSTANT int32_t* table, int64_t head_offset,
                                        int32_t begin, const int32_t* position, int m, int g,
                                        const typename Operand<T>::v8* p, f32x4 (*o)[D / 16]) {
  constexpr int kBits = Format<FMT>::kBits, kRun = Chunk<FMT, D>::kCode / 16;
  constexpr int kEach = COUNT < 8 ? COUNT : 8;
#pragma unroll 1
  for (int t = 0; t < kTile; ++t) {
    const uint32_t lanes = who(t);
    if (!lanes) continue;
    // nothing of this is held in registers while there are no such tokens
    int first = 4 * g, row = m;
    asm volatile("" : "+v"(first), "+v"(row));
    const int32_t j = begin + t;
    const Half h = find_half<FMT, D>(a.pages, head_offset, a.block_shift,
                                     table[j >> a.block_shift], j);
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
      const uint32_t run = first + i;
      const bool here = (lanes >> run) & 1;
#pragma unroll
      for (int at = 0; at < COUNT; at += kEach) {
        Codes<FMT> c = {};
        __builtin_memcpy(c.w, h.v + run * kRun + (FIRST + at) * kBits / 8, kEach * kBits / 8);
        c.byte = static_cast<uint8_t>(h.v_scales[(run * D / 512) << a.block_shift]);
        float x[8];
        c.decode(x);
        __builtin_amdgcn_sched_barrier(0);   // one run at a time: few registers
#pragma unroll
        for (int d = 0; d < kEach; ++d)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float was = o[r][FIRST + at + d][i];
            o[r][FIRST + at + d][i] =
                (here & sees[r]) ? __builtin_fmaf(weight[r], x[d], was) : was;
          }
      }
    }
  }
}

// Which of the tiles that rows [low, high] visit comes v-th.
struct Tiles {
  int32_t first_tiles, skipped, end;
  __device__ __forceinline__ int32_t at(int32_t v) const {
    return v < first_tiles ? v : v + skipped;
  }
};

// Whether every row of [low, high] sees every token of the tile at `begin`.
__device__ __forceinline__ bool seen_whole(const Scope& a, int32_t low, int32_t high,
                                           int32_t begin) {
  return (begin + kTile - 1 <= low) & ((high - begin < a.window) | (begin + kTile <= a.sinks));
}

// Query rows of a 16-row tile as a matrix operand: lane's row, its values [D/4 g, ..).
template <typename T, int D>
__device__ __forceinline__ void load_query(ColdArgs args, ItemPtr it, int32_t row, bool there,
                                           int g, typename Operand<T>::v8* q) {
  const int32_t group = args->group, token = row / group;
  const bool whole_words = args->q.whole_words;
  const T* from = reinterpret_cast<const T*>(args->q.base) +
                  (int64_t(it->token) + token) * args->q.token +
                  (int64_t(it->kv_head) * group + (row - token * group)) * args->q.head +
                  g * (D / 4);
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (there) {
      if (whole_words) {
        const v4u x = *(const gv4u*)(from + s * 8);
        __builtin_memcpy(w, &x, 16);
      } else {
        T t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = from[s * 8 + j];
        __builtin_memcpy(w, t, 16);
      }
    }
    __builtin_memcpy(&q[s], w, 16);
  }
}

// A row's running sums are taken against a score that need not be its largest,
// only near it: 2^kLift stands for `top`, and a probability past kLimit has the
// row's scores looked through for their largest and the sums made before fade
// to it. The types' relative precision is the same over the whole range
// between; looked through for every tile, with the lanes' exchange, it took a
// third of the arithmetic.
// Added to a product of a score of thousands, `lift` is off by as much as it was rounded
// by: nothing beside what rounds such a score, until (past 2^28) it is more than the
// exponents have room for. Rows whose lift passes kLimit take each tile the long
// way, against their largest score itself. So do rows that have no score yet.
// The sum is that of the rounded probabilities, the ones that V is multiplied
// with, as one more product, with ones: what rounding adds to both cancels
// in part (against 64 bits 0.0021 instead of 0.0023 in bfloat16), every lane of a
// row has it, and a matrix instruction does the work of seven additions.
struct RowState {
  float top = -INFINITY;
  float lift = 1e30f;    // kLift - top * c; past kLimit while there is no top
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};   // four times the same
};

// Scores of a row tile (lane's row, eight of its tokens) into probabilities.
template <typename T, int N>
__device__ __forceinline__ typename Operand<T>::v8 softmax_step(const f32x4* x, float c,
                                                               RowState& s, f32x4 (&o)[N]) {
  float e[8];
  const auto exponents = [&](float from, float lift) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i / 4][i % 4] - from, c, lift));
  };
  exponents(0.f, s.lift);
  const float largest =
      fmaxf(fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])),
                  fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7]))), fabsf(s.lift));
  if (__any(largest > Operand<T>::kLimit)) {
    float most = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                       fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    most = fmaxf(s.top, row_max(most));
    const float fade = s.top == most ? 1.f : __builtin_amdgcn_exp2f((s.top - most) * c);
    s.sum *= fade;
#pragma unroll
    for (int d = 0; d < N; ++d) o[d] *= fade;
    s.top = most;
    if (most != -INFINITY) s.lift = Operand<T>::kLift - most * c;
    const bool far = (fabsf(s.lift) > Operand<T>::kLimit) & (most != -INFINITY);
    exponents(far ? most : 0.f, far ? Operand<T>::kLift : s.lift);
  }
  typename Operand<T>::v8 p, ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = static_cast<T>(e[i]);
    ones[i] = T(1.f);
  }
  s.sum = Operand<T>::mma(ones, p, s.sum);
  return p;
}

constexpr int kAttendLanes = 256, kAttendWaves = 4;

// Waves a SIMD has to hold: what the registers allow where 16 rows' sums and two
// tiles of codes take few of them.
template <int D, int R>
constexpr int kAttendPerSimd = D <= 128 && R == 1 ? 3 : D <= 128 ? 2 : 1;
// Tiles on their way. Two, at three waves a SIMD, where the registers hold them:
// with one, at four waves, 48 sequences of 40 heads took 110 us instead of 100.
template <int D, int R>
constexpr int kTilesAhead = R == 1 && D <= 128 ? 2 : 1;

// Where a row's result begins.
template <typename T, typename P>
__device__ __forceinline__ T* result_row(ColdArgs args, P it, int32_t row) {
  const int32_t group = args->group, token = row / group;
  return reinterpret_cast<T*>(args->out.base) + (int64_t(it->token) + token) * args->out.token +
         (int64_t(it->kv_head) * group + (row - token * group)) * args->out.head;
}

// Single tokens and short runs: S^T = K Q^T and O^T = V^T P^T over tiles of 32
// tokens, one pass, with each row's reference score and sum kept as the tiles go by.
// With the tokens along the matrix rows of the first product, its result is the
// second one's operand as it lies in the registers, and a row's state is its
// lane's. Codes become operands in registers (64 conversions and 32 permutes a
// tile of 128-wide heads in mxfp4); the rows of all query heads of a KV head share them.
// Bound by HBM: 64 requests of 8 KV heads (278 MB) take 54 us and their parts 5 to
// join, 4.8 TB/s in all; 48 of 40 heads (536 MB, none cut) 95 us, 5.7 TB/s. What is
// missing to the copy rate of 6.5 is the ends of items (read, join) and the
// scattered kilobyte a block and head.

// Where a workgroup's waves join, a row tile at a time.
template <int D, int R>
struct Joined {
  float part[kAttendWaves][16][D + 4];
  float top[kAttendWaves][16 * R], sum[kAttendWaves][16 * R];
};

template <int FMT, int D, typename T, int R>
__device__ __forceinline__ void attend_item(const Scope& a, ItemPtr it, Joined<D, R>& share) {
  typedef typename Operand<T>::v8 v8;
  constexpr int kSteps = D / 32;    // matrix steps along the head
  constexpr int kOut = D / 16;      // output tiles of 16 values
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, m = lane % 16, g = lane / 16;
  const ColdArgs args = cold_args();
  const auto* table = in_plan<int32_t>(args->plan, args->at_table) + it->table;
  const Tiles tiles = {it->first_tiles, it->window_tile - it->first_tiles, it->tile_end};
  const int64_t head_offset = it->kv_head * Chunk<FMT, D>::bytes(1 << a.block_shift);

  // kAhead tiles are on their way while one is worked on: a tile's K is asked for
  // as soon as the registers it goes to are operands, its V as soon as theirs are,
  // and the blocks that it lies in one step earlier still.
  struct Tile {
    KPart<FMT, D, true> k[2];
    VPart<FMT, D, Chunk<FMT, D>::kCode / 16, true> v;
  };
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
  const auto load_k = [&](Tile& t, const Blocks& b, Half* h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h[i] = find_half<FMT, D>(a.pages, head_offset, a.block_shift, b.block[i],
                               b.position + 16 * i);
      t.k[i].load(h[i], a.block_shift, m, g);
    }
  };
  constexpr int kAhead = kTilesAhead<D, R>;
  Tile held[kAhead];
  int32_t at = it->tile + wave;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (at + i * kAttendWaves < tiles.end) {
      Half h[2];
      load_k(held[i], find(at + i * kAttendWaves), h);
      held[i].v.load(h, a.block_shift, m, g, 0);
    }
  }
  Blocks ahead = find(at + kAhead * kAttendWaves);

  v8 q[R][kSteps];
  int32_t position[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int32_t row = it->row + 16 * r + m;
    const bool there = 16 * r + m < it->rows;
    position[r] = it->base + (there ? row / args->group : 0);
    load_query<T, D>(args, it, row, there, g, q[r]);
  }
  const int32_t low = it->base + it->row / args->group;
  const int32_t high = it->base + (it->row + it->rows - 1) / args->group;

  f32x4 o[R][kOut];
  RowState state[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int d = 0; d < kOut; ++d) o[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const auto step = [&](Tile& t) {
    const int32_t begin = tiles.at(at) * kTile;
    const bool more = at + kAhead * kAttendWaves < tiles.end;

    // scores: lane holds row m, tokens 4g + i of both halves
    f32x4 x[R][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][half] = f32x4{0.f, 0.f, 0.f, 0.f};
      each_constant<0, kSteps>([&](auto s) {
        const v8 k = t.k[half].template operand<T, decltype(s)::value>();
#pragma unroll
        for (int r = 0; r < R; ++r)
          x[r][half] = Operand<T>::mma(k, q[r][decltype(s)::value], x[r][half]);
      });
    }
    Half h[2];
    if (more) load_k(t, ahead, h);
    ahead = find(at + (kAhead + 1) * kAttendWaves);

    // Tokens that some row does not see. All by selection: with branches around
    // the changed elements the compiler lost one of the changes (the first
    // element's, its operands being copied out of the matrix registers in
    // several places).
    uint32_t odd = 0;
    if (!seen_whole(a, low, high, begin) || __any(t.v.template far<T>())) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < R; ++r)
            x[r][half][i] = seen(a, position[r], begin + 16 * half + 4 * g + i) ? x[r][half][i]
                                                                                : -INFINITY;
      odd = t.v.template clear<T>(begin, g, low, high, a.window, a.sinks);
    }

    v8 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) p[r] = softmax_step<T>(x[r], a.c, state[r], o[r]);

    float scale[2][4];
    t.v.scales(scale);
    each_constant<0, kOut / 2>([&](auto b) {
      constexpr int B = decltype(b)::value;
      v8 first, second;
      t.v.template operands<T, B>(scale, &first, &second);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        o[r][2 * B] = Operand<T>::mma(first, p[r], o[r][2 * B]);
        o[r][2 * B + 1] = Operand<T>::mma(second, p[r], o[r][2 * B + 1]);
      }
    });
    if (__any(odd != 0))
      add_far<FMT, D, T, R, 0, kOut>(a, [&](int i) { return lanes_of(odd, i); }, table,
                                     head_offset, begin, position, m, g, p, o);
    if (more) t.v.load(h, a.block_shift, m, g, 0);
    at += kAttendWaves;
  };
  while (at < tiles.end) {
    step(held[0]);
    if constexpr (kAhead == 2) {
      // not by leaving the loop: then the compiler held twenty registers more
      // and spilled some (64 decodes: 71 us instead of 58)
      if (at < tiles.end) step(held[1]);
    }
  }

  // join the waves: each scales its part to the largest of their scores
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float s = state[r].sum[0];
    if (g == 0) {
      share.top[wave][16 * r + m] = state[r].top;
      share.sum[wave][16 * r + m] = s;
    }
  }
  __syncthreads();
  const ColdArgs end_args = cold_args();
  const ItemPtr ended = anew(it);
  constexpr int kRowLanes = 16, kEach = D / kRowLanes;   // of a row, values of each
  const int row = threadIdx.x / kRowLanes, part = threadIdx.x % kRowLanes;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float most = share.top[0][16 * r + m];
#pragma unroll
    for (int w = 1; w < kAttendWaves; ++w) most = fmaxf(most, share.top[w][16 * r + m]);
    const float top = state[r].top;
    const float fade = top == most ? 1.f : __builtin_amdgcn_exp2f((top - most) * a.c);
    float y[kEach] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kOut; ++d)
        share.part[wave][m][(D / 16) * (4 * g + i) + d] = o[r][d][i] * fade;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) y[i] += share.part[w][row][part * kEach + i];
    }
    if (r + 1 < R) __syncthreads();   // before the next row tile's parts
    if (16 * r + row < ended->rows) {
      float all = share.top[0][16 * r + row], total = 0.f;
#pragma unroll
      for (int w = 1; w < kAttendWaves; ++w) all = fmaxf(all, share.top[w][16 * r + row]);
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        const float t = share.top[w][16 * r + row];
        total += share.sum[w][16 * r + row] *
                 (t == all ? 1.f : __builtin_amdgcn_exp2f((t - all) * a.c));
      }
      if (ended->slot < 0) {
        T* to = result_row<T>(end_args, ended, ended->row + 16 * r + row);
        const float inv = 1.f / total;
#pragma unroll
        for (int i = 0; i < kEach; ++i) to[part * kEach + i] = static_cast<T>(y[i] * inv);
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

template <int FMT, int D, typename T, int R>
__global__ __launch_bounds__(kAttendLanes, (kAttendPerSimd<D, R>)) void quant_attend_kernel(
    AttendArgs args) {
  __shared__ Joined<D, R> joined;
  const Scope scope = args.scope;
  const ItemPtr it = in_plan<Item>(args.plan, args.at_items) + blockIdx.x;
  if (static_cast<int32_t>(blockIdx.x) >= in_plan<Header>(args.plan, 0)->items[args.kind]) return;
  attend_item<FMT, D, T, R>(scope, it, joined);
}

// Prompts, as the above: 128 rows a workgroup, 32 a wave. The cache's tokens become matrix
// operands once for all of them: a stage of 64 tokens, each wave making a quarter
// of K's operands and of V's, is laid in shared memory lane by lane as the matrix
// instructions take them, so that reads and writes are whole and without
// conflicts. Two stages: while one is multiplied, the next one's bytes are on their
// way in registers, and one barrier a stage is enough. Four prompts of 1,000 to
// 4,096 tokens, 32 heads over 8 (158 GFLOP) take 218-230 us, 690-725 TFLOP/s; converted
// by every wave for itself, 321. Bound by the issue of two waves a SIMD: 30 % of
// the cycles multiply, 39 % are vector instructions (an exponential, 16
// cycles, for each score); reading operands earlier, waiting for loads elsewhere,
// loads without conditions and wave priorities changed less than 3 %.
constexpr int kStageTiles = 2, kWaveRows = 32;
static_assert(kAttendWaves == 4 && kStageTiles == 2, "a wave makes half a tile's operands");
static_assert(kManyRows == kAttendWaves * kWaveRows, "rows of a workgroup");

template <int D>
struct Stage {
  v4u k[2 * kStageTiles][D / 32][64];
  v4u v[kStageTiles][D / 16][64];
  // tokens that V's operands lack, for each half of a lane's values: whether
  // there are any (by the wave that made them), and then the lanes that cleared them (lanes_of)
  v4u far;
  uint16_t far_lanes[kStageTiles][2][kTile];
};

template <int FMT, int D, typename T>
__device__ __forceinline__ void attend_prompt_item(const Scope& a, ItemPtr it,
                                                   Stage<D> (&stages)[2]) {
  typedef typename Operand<T>::v8 v8;
  constexpr int R = kWaveRows / 16, kSteps = D / 32, kOut = D / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, m = lane % 16, g = lane / 16;
  const ColdArgs args = cold_args();
  const auto* table = in_plan<int32_t>(args->plan, args->at_table) + it->table;
  const Tiles tiles = {it->first_tiles, it->window_tile - it->first_tiles, it->tile_end};
  const int32_t group = args->group;
  const int64_t head_offset = it->kv_head * Chunk<FMT, D>::bytes(1 << a.block_shift);
  const int32_t low = it->base + it->row / group;
  const int32_t high = it->base + (it->row + it->rows - 1) / group;

  // this wave's share of a stage: half a tile of K, half the values of a tile of V
  constexpr int kVBytes = Chunk<FMT, D>::kCode / 32;
  const int own_tile = wave / 2, own_half = wave % 2;
  KPart<FMT, D, false> k;
  VPart<FMT, D, kVBytes, false> v;
  const auto load = [&](int32_t at) {
    if (at + own_tile >= tiles.end) return;
    const int32_t position = tiles.at(at + own_tile) * kTile;
    const Half h[2] = {find_half<FMT, D>(a.pages, head_offset, a.block_shift,
                                         table[position >> a.block_shift], position),
                       find_half<FMT, D>(a.pages, head_offset, a.block_shift,
                                         table[(position + 16) >> a.block_shift], position + 16)};
    k.load(own_half ? h[1] : h[0], a.block_shift, m, g);
    v.load(h, a.block_shift, m, g, own_half * kVBytes);
  };
  const auto lay = [&](Stage<D>& to, int32_t at) {
    uint32_t* const own_far = reinterpret_cast<uint32_t*>(&to.far) + wave;
    if (at + own_tile >= tiles.end) {
      if (lane == 0) *own_far = 0;
      return;
    }
    each_constant<0, kSteps>([&](auto s) {
      const v8 f = k.template operand<T, decltype(s)::value>();
      __builtin_memcpy(&to.k[wave][decltype(s)::value][lane], &f, 16);
    });
    const int32_t begin = tiles.at(at + own_tile) * kTile;
    uint32_t odd = 0;
    if (!seen_whole(a, low, high, begin) || __any(v.template far<T>()))
      odd = v.template clear<T>(begin, g, low, high, a.window, a.sinks);
    const bool far = __any(odd != 0);
    if (lane == 0) *own_far = far;
    if (far) {
      uint32_t lanes = 0;
#pragma unroll 1
      for (int t = 0; t < kTile; ++t) {
        const uint32_t found = lanes_of(odd, t);
        lanes = lane == t ? found : lanes;
      }
      if (lane < kTile) to.far_lanes[own_tile][own_half][lane] = static_cast<uint16_t>(lanes);
    }
    float scale[2][4];
    v.scales(scale);
    each_constant<0, decltype(v)::kPairs>([&](auto b) {
      v8 even, odd;
      v.template operands<T, decltype(b)::value>(scale, &even, &odd);
      const int first = 2 * (own_half * decltype(v)::kPairs + decltype(b)::value);
      __builtin_memcpy(&to.v[own_tile][first][lane], &even, 16);
      __builtin_memcpy(&to.v[own_tile][first + 1][lane], &odd, 16);
    });
  };
  load(it->tile);

  const int32_t row0 = it->row + wave * kWaveRows;
  const int32_t rows = min(max(it->rows - wave * kWaveRows, 0), kWaveRows);
  const int32_t wave_low = it->base + row0 / group;
  const int32_t wave_high = rows ? it->base + (row0 + rows - 1) / group : -1;
  v8 q[R][kSteps];
  int32_t position[R];
  f32x4 o[R][kOut];
  RowState state[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool there = 16 * r + m < rows;
    position[r] = there ? it->base + (row0 + 16 * r + m) / group : wave_low;
    load_query<T, D>(args, it, row0 + 16 * r + m, there, g, q[r]);
#pragma unroll
    for (int d = 0; d < kOut; ++d) o[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const auto multiply = [&](const Stage<D>& from, int32_t at, int tile, uint32_t any_far) {
    if (at + tile >= tiles.end) return;
    const int32_t begin = tiles.at(at + tile) * kTile;
    // tiles that none of the wave's rows sees
    if ((begin > wave_high) |
        ((wave_low - (begin + kTile - 1) >= a.window) & (begin >= a.sinks)))
      return;
    f32x4 x[R][2];
    // The operands are read from shared memory together, V's before the softmax:
    // two at a time where they are used, four prompts took 231 us instead of 226.
    v8 kf[2][kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        __builtin_memcpy(&kf[half][s], &from.k[2 * tile + half][s][lane], 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < R; ++r) x[r][0] = x[r][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < R; ++r) x[r][half] = Operand<T>::mma(kf[half][s], q[r][s], x[r][half]);
    v8 vf[kOut];
#pragma unroll
    for (int d = 0; d < kOut; ++d) __builtin_memcpy(&vf[d], &from.v[tile][d][lane], 16);
    __builtin_amdgcn_sched_barrier(0);
    if (!seen_whole(a, wave_low, wave_high, begin)) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < R; ++r)
            x[r][half][i] = seen(a, position[r], begin + 16 * half + 4 * g + i) ? x[r][half][i]
                                                                                : -INFINITY;
    }
    v8 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) p[r] = softmax_step<T>(x[r], a.c, state[r], o[r]);
#pragma unroll
    for (int d = 0; d < kOut; ++d)
#pragma unroll
      for (int r = 0; r < R; ++r) o[r][d] = Operand<T>::mma(vf[d], p[r], o[r][d]);
    if (!__builtin_amdgcn_readfirstlane(any_far)) return;
    const auto add = [&](auto half) {
      constexpr int kHalf = decltype(half)::value;
      if (!__builtin_amdgcn_readfirstlane(uint32_t{from.far[2 * tile + kHalf]})) return;
      add_far<FMT, D, T, R, kHalf * kOut / 2, kOut / 2>(
          a, [&](int t) {
            return __builtin_amdgcn_readfirstlane(uint32_t{from.far_lanes[tile][kHalf][t]});
          }, table, head_offset, begin, position, m, g, p, o);
    };
    add(std::integral_constant<int, 0>{});
    add(std::integral_constant<int, 1>{});
  };

  int turn = 0;
  for (int32_t at = it->tile; at < tiles.end; at += kStageTiles, turn ^= 1) {
    lay(stages[turn], at);
    load(at + kStageTiles);
    __syncthreads();
    const v4u far = stages[turn].far;
    const uint32_t any_far = far[0] | far[1] | far[2] | far[3];
#pragma unroll
    for (int tile = 0; tile < kStageTiles; ++tile) multiply(stages[turn], at, tile, any_far);
  }

  const ColdArgs end_args = cold_args();
  const ItemPtr ended = anew(it);
  const int32_t slot = ended->slot;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float total = state[r].sum[0];
    const int32_t n = row0 + 16 * r + m;
    if (16 * r + m >= rows) continue;
    float* part = end_args->work + slot * end_args->slot_floats + (n - ended->row) * (D + 4);
    T* to = result_row<T>(end_args, ended, n);
    const float inv = slot < 0 ? 1.f / total : 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[kOut];
#pragma unroll
      for (int d = 0; d < kOut; ++d) y[d] = o[r][d][i] * inv;
      const int first = kOut * (4 * g + i);
      if (slot >= 0) {
#pragma unroll
        for (int d = 0; d < kOut; d += 4) __builtin_memcpy(part + first + d, y + d, 16);
      } else {
        T t[kOut];
#pragma unroll
        for (int d = 0; d < kOut; ++d) t[d] = static_cast<T>(y[d]);
        if (end_args->out.whole_words) {
          __builtin_memcpy(__builtin_assume_aligned(to + first, kOut < 8 ? 8 : 16), t, sizeof t);
        } else {
#pragma unroll
          for (int d = 0; d < kOut; ++d) to[first + d] = t[d];
        }
      }
    }
    if (slot >= 0 && g == 0) {
      part[D] = state[r].top;
      part[D + 1] = total;
    }
  }
}

template <int FMT, int D, typename T>
__global__ __launch_bounds__(kAttendLanes, D == 256 ? 1 : 2) void quant_prompt_kernel(
    AttendArgs args) {
  __shared__ Stage<D> stages[2];
  const Scope scope = args.scope;
  const ItemPtr it = in_plan<Item>(args.plan, args.at_items) + blockIdx.x;
  if (static_cast<int32_t>(blockIdx.x) >= in_plan<Header>(args.plan, 0)->items[args.kind]) return;
  attend_prompt_item<FMT, D, T>(scope, it, stages);
}

// Rows whose tiles several items shared: their parts, scaled to the largest
// score of all, over the sum of their sums. A workgroup's lanes are groups of D / 4,
// four values a lane. Of up to kMergeRows parts each group takes rows of its own;
// more (few rows over a long axis) are shared out to the groups, one row a workgroup.
// 5 us, most of it the launch and two dependent reads; when one lane a value
// walked all parts, 128 parts of 56 rows took 54.
template <int D, typename T>
__global__ __launch_bounds__(256) void quant_merge_kernel(AttendArgs a) {
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
  const auto store = [&](int32_t row, f32x4 y, float total) {
    T* to = result_row<T>((ColdArgs)__builtin_amdgcn_kernarg_segment_ptr(), mg, mg->row + row) +
            4 * at;
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = static_cast<T>(y[i] / total);
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
        const float fade = t[p] == most ? 1.f : __builtin_amdgcn_exp2f((t[p] - most) * a.scope.c);
        y += *reinterpret_cast<const f32x4*>(from + p * each + 4 * at) * fade;
        total += from[p * each + D + 1] * fade;
      }
      store(row, y, total);
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
    const float fade = t == most ? 1.f : __builtin_amdgcn_exp2f((t - most) * a.scope.c);
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
  store(0, y, total);
}

}  // namespace

#endif  // AEGKV_QUANT_CACHE_H
