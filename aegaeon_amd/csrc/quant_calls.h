// Entry points over a quantised cache (include/aegkv.h): checks, then launches
// of the kernels of quant_cache.h. Part of aegkv.hip's translation unit.
#ifndef AEGKV_QUANT_CALLS_H
#define AEGKV_QUANT_CALLS_H

#include "quant_cache.h"
#include "value_places.h"

#include <initializer_list>

namespace {

struct QuantCall {
  Header h;
  const char* plan;      // on the device
  const char* k;
  const char* v;
  int64_t page_bytes;
  int format, head_dim;
  bool capturing;
};

int64_t quant_page_bytes(int format, int32_t block_size, int32_t kv_heads, int32_t head_dim) {
  const int64_t code = int64_t(head_dim) * (format == AEGKV_FORMAT_MXFP4 ? 4 : 8) / 8;
  return int64_t(kv_heads) * block_size * (code + head_dim / 32);
}

int check_quant_shape(int format, int32_t head_dim) {
  if (format != AEGKV_FORMAT_MXFP4 && format != AEGKV_FORMAT_MXFP8)
    return fail(AEGKV_EINVAL, "unknown cache format %d", format);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(AEGKV_EINVAL, "heads are 64, 128 or 256 values wide, not %d", head_dim);
  return 0;
}

int read_header(const void* plan, Header* h) {
  if (!plan) return fail(AEGKV_EINVAL, "plan must not be null");
  std::memcpy(h, plan, sizeof *h);
  if (h->magic != kMagic) return fail(AEGKV_EINVAL, "this is no plan of aegkv_batch_plan");
  return 0;
}

int open_call(const void* plan, const void* device_plan, int format, int32_t head_dim,
              const void* k_pages, const void* v_pages, hipStream_t stream, QuantCall* c) {
  g_err[0] = '\0';
  int rc = check_quant_shape(format, head_dim);
  if (rc) return rc;
  rc = read_header(plan, &c->h);
  if (rc) return rc;
  const Header& h = c->h;
  c->plan = static_cast<const char*>(device_plan);
  c->k = static_cast<const char*>(k_pages);
  c->v = static_cast<const char*>(v_pages);
  c->format = format;
  c->head_dim = head_dim;
  c->page_bytes = quant_page_bytes(format, h.block_size, h.kv_heads, head_dim);
  if (!device_plan || !k_pages || !v_pages)
    return fail(AEGKV_EINVAL, "the plan's device copy and both caches must not be null");
  if (!aligned16(device_plan) || !aligned16(k_pages) || !aligned16(v_pages))
    return fail(AEGKV_EINVAL, "the plan's device copy and the caches must be 16-byte aligned");
  rc = check_device_range(device_plan, h.room.bytes, "the plan's device copy");
  if (!rc) rc = check_device_range(k_pages, h.num_blocks * c->page_bytes, "the K cache");
  if (!rc) rc = check_device_range(v_pages, h.num_blocks * c->page_bytes, "the V cache");
  if (rc) return rc;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  AEGKV_HIP(hipStreamIsCapturing(stream, &status));
  c->capturing = status != hipStreamCaptureStatusNone;
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

Named k_cache(const QuantCall& c) {
  return Named{place(c.k, c.h.num_blocks * c.page_bytes), "the K cache"};
}
Named v_cache(const QuantCall& c) {
  return Named{place(c.v, c.h.num_blocks * c.page_bytes), "the V cache"};
}
Named plan_place(const QuantCall& c) {
  return Named{place(c.plan, c.h.room.bytes), "the plan's device copy"};
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

template <typename F>
int by_shape(int format, int head_dim, const F& f) {
  const auto width = [&](auto fmt) {
    switch (head_dim) {
      case 64: return f(fmt, Constant<64>{});
      case 128: return f(fmt, Constant<128>{});
      default: return f(fmt, Constant<256>{});
    }
  };
  return format == AEGKV_FORMAT_MXFP4 ? width(Constant<AEGKV_FORMAT_MXFP4>{})
                                      : width(Constant<AEGKV_FORMAT_MXFP8>{});
}

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

// Rows (a token of a head) that a workgroup of a write or read takes about: all
// heads of a decode step's single tokens, a few of whole spans.
constexpr int64_t kSpanRows = 64;

int span_args(const QuantCall& c, bool fresh, SpanArgs* a, dim3* grid) {
  const Header& h = c.h;
  const int64_t spans = fresh ? h.room.new_spans : h.room.read_spans;
  const int64_t tokens = fresh ? h.room.tokens : spans * kSpan;
  a->plan = c.plan;
  a->at_seqs = h.room.at_seqs;
  a->at_table = h.room.at_table;
  a->at_new_spans = h.room.at_new_spans;
  a->pages[0] = const_cast<char*>(c.k);
  a->pages[1] = const_cast<char*>(c.v);
  a->page_bytes = c.page_bytes;
  a->kv_heads = h.kv_heads;
  a->block_size = h.block_size;
  a->fresh = fresh;
  const int64_t heads = kSpanRows * spans / std::max<int64_t>(1, tokens);
  a->heads_each =
      static_cast<int32_t>(std::min<int64_t>(h.kv_heads, std::max<int64_t>(1, heads)));
  a->head_groups = (h.kv_heads + a->heads_each - 1) / a->heads_each;
  *grid = dim3(static_cast<uint32_t>(spans * a->head_groups), 2);
  return check_grid(spans * a->head_groups, kSpanLanes);
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

extern "C" {

int aegkv_quant_page_bytes(int format, int32_t block_size, int32_t kv_heads, int32_t head_dim,
                           int64_t* bytes) {
  g_err[0] = '\0';
  if (!bytes) return fail(AEGKV_EINVAL, "bytes must not be null");
  Header h;
  int rc = check_quant_shape(format, head_dim);
  if (rc) return rc;
  rc = describe(h, 1, block_size, kv_heads, kv_heads, 0, 0);
  if (rc) return rc;
  *bytes = quant_page_bytes(format, block_size, kv_heads, head_dim);
  return 0;
}

int aegkv_quant_write(const void* plan, const void* device_plan, int format, int32_t head_dim,
                      void* k_pages, void* v_pages, const void* k, int64_t k_token_stride,
                      int64_t k_head_stride, const void* v, int64_t v_token_stride,
                      int64_t v_head_stride, int64_t num_tokens, int dtype, hipStream_t stream) {
  QuantCall c;
  int rc = open_call(plan, device_plan, format, head_dim, k_pages, v_pages, stream, &c);
  if (rc) return rc;
  rc = check_apart(k_cache(c), {v_cache(c), plan_place(c)});
  if (!rc) rc = check_apart(v_cache(c), {plan_place(c)});
  if (rc) return rc;
  rc = check_count(num_tokens, c.h.num_tokens, c.h.room.tokens, c.capturing, "k and v");
  SpanArgs a;
  dim3 grid;
  if (!rc) rc = check_values(k, num_tokens, c.h.kv_heads, head_dim, dtype, k_token_stride,
                             k_head_stride, false, "k", &a.values[0]);
  if (!rc) rc = check_values(v, num_tokens, c.h.kv_heads, head_dim, dtype, v_token_stride,
                             v_head_stride, false, "v", &a.values[1]);
  const int64_t reached = c.capturing ? c.h.room.tokens : c.h.num_tokens;
  for (int i = 0; i < 2 && !rc; ++i)
    rc = check_apart(Named{rows_place(a.values[i], reached, c.h.kv_heads, head_dim, dtype),
                           i ? "v" : "k"}, {k_cache(c), v_cache(c)});
  if (!rc) rc = span_args(c, true, &a, &grid);
  if (rc || grid.x == 0) return rc;
  return by_shape(format, head_dim, [&](auto fmt, auto d) {
    return by_type(dtype, [&](auto t) {
      return launch(quant_write_kernel<decltype(fmt)::value, decltype(d)::value, decltype(t)>, grid,
                    kSpanLanes, stream, a, "quant_write_kernel launch");
    });
  });
}

int aegkv_quant_read(const void* plan, const void* device_plan, int format, int32_t head_dim,
                     const void* k_pages, const void* v_pages, int new_tokens, void* k,
                     int64_t k_token_stride, int64_t k_head_stride, void* v,
                     int64_t v_token_stride, int64_t v_head_stride, int64_t num_tokens, int dtype,
                     hipStream_t stream) {
  QuantCall c;
  int rc = open_call(plan, device_plan, format, head_dim, k_pages, v_pages, stream, &c);
  if (rc) return rc;
  const Header& h = c.h;
  if (!new_tokens && !h.complete)
    return fail(AEGKV_ERANGE, "some columns of the batch are released: their tokens are gone");
  rc = new_tokens
           ? check_count(num_tokens, h.num_tokens, h.room.tokens, c.capturing, "k and v")
           : check_count(num_tokens, h.read_tokens, h.room.read_spans * kSpan, c.capturing,
                         "k and v");
  SpanArgs a;
  dim3 grid;
  if (!rc) rc = check_values(k, num_tokens, h.kv_heads, head_dim, dtype, k_token_stride,
                             k_head_stride, true, "k", &a.values[0]);
  if (!rc) rc = check_values(v, num_tokens, h.kv_heads, head_dim, dtype, v_token_stride,
                             v_head_stride, true, "v", &a.values[1]);
  if (!rc) {
    const int64_t reached = new_tokens ? (c.capturing ? h.room.tokens : h.num_tokens)
                                       : (c.capturing ? h.room.read_spans * kSpan : h.read_tokens);
    const Place to[2] = {rows_place(a.values[0], reached, h.kv_heads, head_dim, dtype),
                         rows_place(a.values[1], reached, h.kv_heads, head_dim, dtype)};
    rc = check_apart(Named{to[0], "k"}, {Named{to[1], "v"}, k_cache(c), v_cache(c),
                                         plan_place(c)});
    if (!rc) rc = check_apart(Named{to[1], "v"}, {k_cache(c), v_cache(c), plan_place(c)});
  }
  if (!rc) rc = span_args(c, new_tokens != 0, &a, &grid);
  if (rc || grid.x == 0) return rc;
  return by_shape(format, head_dim, [&](auto fmt, auto d) {
    return by_type(dtype, [&](auto t) {
      return launch(quant_read_kernel<decltype(fmt)::value, decltype(d)::value, decltype(t)>, grid,
                    kSpanLanes, stream, a, "quant_read_kernel launch");
    });
  });
}

int aegkv_quant_attend_workspace(const void* plan, int32_t head_dim, int64_t* bytes) {
  g_err[0] = '\0';
  Header h;
  if (!bytes) return fail(AEGKV_EINVAL, "bytes must not be null");
  int rc = read_header(plan, &h);
  if (!rc) rc = check_quant_shape(AEGKV_FORMAT_MXFP4, head_dim);
  if (rc) return rc;
  int64_t at[kKinds], each[kKinds];
  *bytes = 4 * parts_floats(h, head_dim, at, each);
  return 0;
}

int aegkv_quant_attend(const void* plan, const void* device_plan, int format, int32_t head_dim,
                       const void* k_pages, const void* v_pages, const void* q,
                       int64_t q_token_stride, int64_t q_head_stride, void* out,
                       int64_t out_token_stride, int64_t out_head_stride, int64_t num_tokens,
                       int dtype, double scale, void* workspace, int64_t workspace_bytes,
                       hipStream_t stream) {
  QuantCall c;
  int rc = open_call(plan, device_plan, format, head_dim, k_pages, v_pages, stream, &c);
  if (rc) return rc;
  const Header& h = c.h;
  if (dtype != AEGKV_DTYPE_BFLOAT16 && dtype != AEGKV_DTYPE_FLOAT16)
    return fail(AEGKV_EINVAL, "queries are bfloat16 or float16, not type %d", dtype);
  const double factor = scale * 1.4426950408889634;
  if (!(scale > 0) || !(factor < 3e38) || !(factor > 1e-37))
    return fail(AEGKV_EINVAL, "scale %g is not a positive number", scale);
  rc = check_count(num_tokens, h.num_tokens, h.room.tokens, c.capturing, "q and out");
  AttendArgs a;
  if (!rc) rc = check_values(q, num_tokens, h.heads, head_dim, dtype, q_token_stride,
                             q_head_stride, false, "q", &a.q);
  if (!rc) rc = check_values(out, num_tokens, h.heads, head_dim, dtype, out_token_stride,
                             out_head_stride, true, "out", &a.out);
  if (rc) return rc;
  const int64_t floats = parts_floats(h, head_dim, a.kind_work, a.kind_slot_floats);
  if (floats) {
    if (!workspace || !aligned16(workspace) || workspace_bytes < 4 * floats)
      return fail(AEGKV_ENOMEM, "attention over this plan takes a workspace of %lld bytes, "
                  "16-byte aligned", ll(4 * floats));
    rc = check_device_range(workspace, 4 * floats, "the workspace");
    if (rc) return rc;
  }
  const int64_t reached = c.capturing ? h.room.tokens : h.num_tokens;
  const Place from = rows_place(a.q, reached, h.heads, head_dim, dtype);
  const Place to = rows_place(a.out, reached, h.heads, head_dim, dtype);
  const Place parts = place(workspace, 4 * floats);
  // in place every row is read by the workgroup that writes it, or before all that do
  if (!same(from, to)) rc = check_apart(Named{to, "out"}, {Named{from, "q"}});
  if (!rc) rc = check_apart(Named{to, "out"}, {k_cache(c), v_cache(c), plan_place(c)});
  if (!rc) rc = check_apart(Named{parts, "the workspace"},
                            {Named{to, "out"}, Named{from, "q"}, k_cache(c), v_cache(c),
                             plan_place(c)});
  if (rc) return rc;
  a.plan = c.plan;
  a.at_table = h.room.at_table;
  a.at_merges = h.room.at_merges;
  a.scope.pages = QuantPages{c.k, c.v, c.page_bytes};
  a.work_base = static_cast<float*>(workspace);
  a.scope.c = static_cast<float>(factor);
  a.scope.block_shift = __builtin_ctz(h.block_size);
  a.group = h.group;
  a.scope.window = h.window ? h.window : INT32_MAX;
  a.scope.sinks = h.sinks;
  rc = check_grid(h.room.merges, 256);
  for (int kind = 0; kind < kKinds && !rc; ++kind)
    rc = check_grid(h.room.items[kind], kAttendLanes);
  if (rc) return rc;
  return by_shape(format, head_dim, [&](auto fmt, auto d) {
    constexpr int kFormat = decltype(fmt)::value, kDim = decltype(d)::value;
    const auto attend = [&](auto t) {
      typedef decltype(t) T;
      for (int kind = 0; kind < kKinds; ++kind) {
        if (!h.room.items[kind]) continue;
        a.kind = kind;
        a.at_items = h.room.at_items[kind];
        a.work = a.work_base + a.kind_work[kind];
        a.slot_floats = a.kind_slot_floats[kind];
        const dim3 grid(static_cast<uint32_t>(h.room.items[kind]));
        const auto kernel = kind == kFew    ? quant_attend_kernel<kFormat, kDim, T, 1>
                            : kind == kMore ? quant_attend_kernel<kFormat, kDim, T, 2>
                                            : quant_prompt_kernel<kFormat, kDim, T>;
        const int rc = launch(kernel, grid, kAttendLanes, stream, a, "quant_attend_kernel launch");
        if (rc) return rc;
      }
      if (h.room.merges)
        return launch(quant_merge_kernel<kDim, T>, dim3(static_cast<uint32_t>(h.room.merges)), 256,
                      stream, a, "quant_merge_kernel launch");
      return 0;
    };
    return dtype == AEGKV_DTYPE_BFLOAT16 ? attend(__bf16{}) : attend(_Float16{});
  });
}

}  // extern "C"

#endif  // AEGKV_QUANT_CALLS_H
