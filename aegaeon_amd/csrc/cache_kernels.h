// What the kernels over paged caches share: access to the plan, rows of values,
// matrix operands, and what a query sees. Device code; internal to the library.
#ifndef AEGKV_CACHE_KERNELS_H
#define AEGKV_CACHE_KERNELS_H

#include <hip/hip_runtime.h>

#include "batch_plan.h"

#include <cstdint>
#include <type_traits>

namespace {

using namespace aegkv_batch;

typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) v4u gv4u;  // global (VM) address space
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

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

// Matrix operands: eight values of a lane. kLift, kLimit: see RowState (softmax
// sums against a reference score).
template <typename T>
struct Matrix;
template <>
struct Matrix<__bf16> {
  typedef bf16x8 v8;
  static constexpr float kLift = 0.f, kLimit = 65536.f;
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Matrix<_Float16> {
  typedef f16x8 v8;
  // float16 keeps 2^-24 at the least and 2^16 at the most: lifted, small
  // probabilities of long contexts are not lost beside the largest one (the sum
  // is lifted alike), and a row may still grow 2^8-fold
  static constexpr float kLift = 7.f, kLimit = 32768.f;
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

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

// How scores are scaled and what of the cache a query sees.
struct Sight {
  float c;              // scale * log2(e)
  int32_t block_shift, window, sinks;
};

// Whether a query at position p sees position j (window: INT32_MAX for none).
__device__ __forceinline__ bool seen(const Sight& a, int32_t p, int32_t j) {
  return (j <= p) & ((p - j < a.window) | (j < a.sinks));
}

// Which of the tiles that rows [low, high] visit comes v-th.
struct Tiles {
  int32_t first_tiles, skipped, end;
  __device__ __forceinline__ int32_t at(int32_t v) const {
    return v < first_tiles ? v : v + skipped;
  }
};

// Whether every row of [low, high] sees every token of the tile at `begin`.
__device__ __forceinline__ bool seen_whole(const Sight& a, int32_t low, int32_t high,
                                           int32_t begin) {
  return (begin + kTile - 1 <= low) & ((high - begin < a.window) | (begin + kTile <= a.sinks));
}

// The tokens of `odd` (a lane's bits, as VPart::clear gives them): bit m for token t of the
// tile where lane m of its four tokens' has it.
__device__ __forceinline__ uint32_t lanes_of(uint32_t odd, int t) {
  const uint64_t all = __ballot((odd >> (4 * (t / 16) + t % 4)) & 1);
  return static_cast<uint32_t>(all >> (16 * (t % 16 / 4))) & 0xFFFFu;
}

}  // namespace

#endif  // AEGKV_CACHE_KERNELS_H
