// What the entry points over paged caches share: checks of their arguments, and
// launches. Part of aegkv.hip's translation unit, whose checks of device memory and
// error texts it uses.
#ifndef AEGKV_CACHE_CALLS_H
#define AEGKV_CACHE_CALLS_H

#include "cache_kernels.h"
#include "value_places.h"

#include <initializer_list>

namespace {

int read_header(const void* plan, Header* h) {
  if (!plan) return fail(AEGKV_EINVAL, "plan must not be null");
  std::memcpy(h, plan, sizeof *h);
  if (h->magic != kMagic) return fail(AEGKV_EINVAL, "this is no plan of aegkv_batch_plan");
  return 0;
}

int element_bytes(int dtype) {
  return dtype == AEGKV_DTYPE_FLOAT32 ? 4
         : dtype == AEGKV_DTYPE_BFLOAT16 || dtype == AEGKV_DTYPE_FLOAT16 ? 2 : 0;
}

// [tokens][heads][head_dim] at `base`; `written`: no two values share a place.
int check_values(const void* base, int64_t tokens, int32_t heads, int32_t head_dim, int dtype,
                 int64_t token_stride, int64_t head_stride, bool written, const char* what,
                 Values* out) {
  const int es = element_bytes(dtype);
  if (!es) return fail(AEGKV_EINVAL, "%s: unknown type %d", what, dtype);
  *out = Values{static_cast<char*>(const_cast<void*>(base)), token_stride, head_stride, false};
  if (tokens == 0) return 0;
  if (!base) return fail(AEGKV_EINVAL, "%s must not be null", what);
  constexpr int64_t kMost = int64_t(1) << 40;
  if (token_stride < 0 || head_stride < 0 || token_stride > kMost || head_stride > kMost)
    return fail(AEGKV_EINVAL, "%s: strides %lld and %lld", what, ll(token_stride),
                ll(head_stride));
  if (reinterpret_cast<uintptr_t>(base) % es)
    return fail(AEGKV_EINVAL, "%s must be aligned to its %d-byte elements", what, es);
  const __int128 last = static_cast<__int128>(tokens - 1) * token_stride +
                        static_cast<__int128>(heads - 1) * head_stride + head_dim;
  if (last > (static_cast<__int128>(1) << 46))
    return fail(AEGKV_ERANGE, "%s is larger than any device", what);
  if (written) {
    const __int128 by_token = static_cast<__int128>(heads - 1) * head_stride + head_dim;
    const __int128 by_head = static_cast<__int128>(tokens - 1) * token_stride + head_dim;
    const bool heads_apart = heads == 1 || head_stride >= head_dim;
    const bool tokens_apart = tokens == 1 || token_stride >= head_dim;
    if (!heads_apart || !tokens_apart ||
        (heads > 1 && tokens > 1 && token_stride < by_token && head_stride < by_head))
      return fail(AEGKV_EOVERLAP, "%s: rows of %d values overlap at strides %lld and %lld", what,
                  head_dim, ll(token_stride), ll(head_stride));
  }
  out->whole_words =
      aligned16(base) && (token_stride * es) % 16 == 0 && (head_stride * es) % 16 == 0;
  return check_device_range(base, static_cast<int64_t>(last) * es, what);
}

// Values that a call takes: those of the plan's tokens, or in a captured call,
// which a replay after an update may ask for more, of all it has room for.
int check_count(int64_t given, int64_t now, int64_t room, bool capturing, const char* what) {
  const int64_t need = capturing ? room : now;
  if (given < need)
    return fail(AEGKV_ERANGE, "%s holds %lld tokens of %lld%s", what, ll(given), ll(need),
                capturing ? " that a replay may reach" : "");
  return 0;
}

// The first `tokens` rows of checked values.
Place rows_place(const Values& v, int64_t tokens, int32_t heads, int32_t head_dim, int dtype) {
  const int64_t es = element_bytes(dtype);
  return place(v.base, tokens, heads, head_dim * es, v.token * es, v.head * es);
}

// What a call writes shares no byte with what it reads beside it: workgroups run
// in no order.
struct Named {
  Place at;
  const char* what;
};

int check_apart(const Named& w, std::initializer_list<Named> others) {
  for (const Named& o : others)
    if (overlap(w.at, o.at)) return fail(AEGKV_EOVERLAP, "%s and %s overlap", w.what, o.what);
  return 0;
}

template <typename F>
int by_type(int dtype, const F& f) {
  switch (dtype) {
    case AEGKV_DTYPE_BFLOAT16: return f(__bf16{});
    case AEGKV_DTYPE_FLOAT16: return f(_Float16{});
    default: return f(float{});
  }
}

template <int V>
struct Constant {
  static constexpr int value = V;
};

template <typename K, typename A>
int launch(K kernel, dim3 grid, int lanes, hipStream_t stream, const A& args, const char* what) {
  (void)hipGetLastError();  // clear a stale error: the check below is for this launch
  kernel<<<grid, lanes, 0, stream>>>(args);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_fail(e, what);
}

// Work items of a dispatch are counted in 32 bits along an axis.
int check_grid(int64_t workgroups, int lanes) {
  if (workgroups > (int64_t(1) << 32) / lanes - 1)
    return fail(AEGKV_ENOMEM, "%lld workgroups are more than one launch holds", ll(workgroups));
  return 0;
}

// Workspace of attention: each kind's parts one after another.
int64_t parts_floats(const Header& h, int32_t head_dim, int64_t* at, int64_t* each) {
  int64_t floats = 0;
  for (int kind = 0; kind < kKinds; ++kind) {
    at[kind] = floats;
    each[kind] = int64_t(kKindRows[kind]) * (head_dim + 4);   // row, its top and sum
    floats += h.room.slots[kind] * each[kind];
  }
  return floats;
}

}  // namespace

#endif  // AEGKV_CACHE_CALLS_H
