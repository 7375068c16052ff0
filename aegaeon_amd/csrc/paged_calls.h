// Entry points over an ordinary paged cache (include/aegkv.h): checks, then
// launches of the kernels of paged_cache.h. Part of aegkv.hip's translation unit.
#ifndef AEGKV_PAGED_CALLS_H
#define AEGKV_PAGED_CALLS_H

#include "cache_calls.h"
#include "paged_cache.h"

#include <vector>

namespace {

struct PagedCall {
  Header h;
  const char* plan;      // on the device
  aegkv_paged_cache cache;
  Pages pages;
  int64_t page_bytes;
  bool capturing;
};

int is_capturing(hipStream_t stream, bool* capturing) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  AEGKV_HIP(hipStreamIsCapturing(stream, &status));
  *capturing = status != hipStreamCaptureStatusNone;
  return 0;
}

Place pages_place(const void* base, const PagedCall& c, int64_t block_bytes) {
  return place(base, c.h.num_blocks, 1, c.page_bytes, block_bytes, 0);
}
Named k_cache(const PagedCall& c) {
  return Named{pages_place(c.cache.k_pages, c, c.cache.k_block_bytes), "the K cache"};
}
Named v_cache(const PagedCall& c) {
  return Named{pages_place(c.cache.v_pages, c, c.cache.v_block_bytes), "the V cache"};
}
Named plan_place(const PagedCall& c) {
  return Named{place(c.plan, c.h.room.bytes), "the plan's device copy"};
}

int check_plan(const void* plan, const void* device_plan, Header* h) {
  const int rc = read_header(plan, h);
  if (rc) return rc;
  if (!device_plan || !aligned16(device_plan))
    return fail(AEGKV_EINVAL, "the plan's device copy must not be null, and 16-byte aligned");
  return check_device_range(device_plan, h->room.bytes, "the plan's device copy");
}

int open_paged(const void* plan, const void* device_plan, const aegkv_paged_cache* cache,
               hipStream_t stream, PagedCall* c) {
  g_err[0] = '\0';
  if (!cache) return fail(AEGKV_EINVAL, "cache must not be null");
  int rc = check_plan(plan, device_plan, &c->h);
  if (rc) return rc;
  const Header& h = c->h;
  c->plan = static_cast<const char*>(device_plan);
  c->cache = *cache;
  if (cache->dtype != AEGKV_DTYPE_BFLOAT16 && cache->dtype != AEGKV_DTYPE_FLOAT16)
    return fail(AEGKV_EINVAL, "a cache holds bfloat16 or float16, not type %d", cache->dtype);
  if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256)
    return fail(AEGKV_EINVAL, "heads are 64, 128 or 256 values wide, not %d", cache->head_dim);
  if (cache->block_size != h.block_size || cache->kv_heads != h.kv_heads)
    return fail(AEGKV_EINVAL, "a plan of %d-token blocks and %d KV heads over a cache of %d and %d",
                h.block_size, h.kv_heads, cache->block_size, cache->kv_heads);
  if (cache->num_blocks < h.num_blocks)
    return fail(AEGKV_ERANGE, "a plan over %lld blocks, a cache of %lld", ll(h.num_blocks),
                ll(cache->num_blocks));
  const int64_t head_bytes = 2 * int64_t(cache->head_dim);
  c->page_bytes = head_bytes * h.kv_heads * h.block_size;
  // offsets inside a page are 32-bit
  if (c->page_bytes > (int64_t(1) << 30))
    return fail(AEGKV_EINVAL, "a page of %lld bytes is too large", ll(c->page_bytes));
  const char* const names[2] = {"the K cache", "the V cache"};
  const void* const bases[2] = {cache->k_pages, cache->v_pages};
  const int64_t strides[2] = {cache->k_block_bytes, cache->v_block_bytes};
  for (int i = 0; i < 2; ++i) {
    if (!bases[i] || !aligned16(bases[i]) || strides[i] % 16)
      return fail(AEGKV_EINVAL, "%s must not be null, and its blocks 16-byte aligned", names[i]);
    if (strides[i] < c->page_bytes || strides[i] > (int64_t(1) << 40))
      return fail(AEGKV_EINVAL, "%s: blocks of %lld bytes, %lld apart", names[i],
                  ll(c->page_bytes), ll(strides[i]));
    const __int128 bytes = static_cast<__int128>(h.num_blocks - 1) * strides[i] + c->page_bytes;
    if (bytes > (static_cast<__int128>(1) << 46))
      return fail(AEGKV_ERANGE, "%s is larger than any device", names[i]);
    rc = check_device_range(bases[i], static_cast<int64_t>(bytes), names[i]);
    if (rc) return rc;
  }
  c->pages.k = static_cast<const char*>(cache->k_pages);
  c->pages.v = static_cast<const char*>(cache->v_pages);
  c->pages.k_block = cache->k_block_bytes;
  c->pages.v_block = cache->v_block_bytes;
  c->pages.token = static_cast<int32_t>(cache->head_major ? head_bytes : head_bytes * h.kv_heads);
  c->pages.head = static_cast<int32_t>(cache->head_major ? head_bytes * h.block_size : head_bytes);
  return is_capturing(stream, &c->capturing);
}

Sight sight_of(const Header& h, float c) {
  Sight s;
  s.c = c;
  s.block_shift = __builtin_ctz(h.block_size);
  s.window = h.window ? h.window : INT32_MAX;
  s.sinks = h.sinks;
  return s;
}

int check_scale(double scale, float* c) {
  const double factor = scale * 1.4426950408889634;
  if (!(scale > 0) || !(factor < 3e38) || !(factor > 1e-37))
    return fail(AEGKV_EINVAL, "scale %g is not a positive number", scale);
  *c = static_cast<float>(factor);
  return 0;
}

// Rows of a call: of `heads` heads and a type, at least `now` of them (`room` in a capture).
int check_rows(const aegkv_rows* rows, int32_t heads, int32_t head_dim, int dtype, int64_t now,
               int64_t room, bool capturing, bool written, const char* what, Values* out) {
  if (!rows) return fail(AEGKV_EINVAL, "%s must not be null", what);
  if (rows->heads != heads)
    return fail(AEGKV_EINVAL, "%s: %d heads, not %d", what, rows->heads, heads);
  if (rows->dtype != dtype)
    return fail(AEGKV_EINVAL, "%s: type %d, not %d", what, rows->dtype, dtype);
  const int rc = check_count(rows->tokens, now, room, capturing, what);
  if (rc) return rc;
  return check_values(rows->base, rows->tokens, heads, head_dim, dtype, rows->token_stride,
                      rows->head_stride, written, what, out);
}

int64_t reached(const PagedCall& c) { return c.capturing ? c.h.room.tokens : c.h.num_tokens; }

Named rows_named(const Values& v, int64_t tokens, int32_t heads, int32_t head_dim, int dtype,
                 const char* what) {
  return Named{rows_place(v, tokens, heads, head_dim, dtype), what};
}

int check_rotary(const aegkv_rotary* r, int32_t head_dim, PlaceArgs* a) {
  if (r->dim < 2 || r->dim > head_dim || r->dim % 2)
    return fail(AEGKV_EINVAL, "%d rotated values of a head of %d", r->dim, head_dim);
  if (!r->turns || reinterpret_cast<uintptr_t>(r->turns) % 8)
    return fail(AEGKV_EINVAL, "turns must not be null, and 8-byte aligned");
  a->turns = r->turns;
  a->pairs = r->dim / 2;
  a->interleaved = r->interleaved != 0;
  a->amplitude = static_cast<float>(r->amplitude);
  return check_device_range(r->turns, int64_t(a->pairs) * 8, "turns");
}

int check_positions(const void* positions, int64_t given, int position_bytes, int64_t need,
                    PlaceArgs* a) {
  if (position_bytes != 4 && position_bytes != 8)
    return fail(AEGKV_EINVAL, "positions of %d bytes", position_bytes);
  if (given < need)
    return fail(AEGKV_ERANGE, "%lld positions of %lld tokens", ll(given), ll(need));
  if (reinterpret_cast<uintptr_t>(positions) % position_bytes)
    return fail(AEGKV_EINVAL, "positions must be aligned to their %d bytes", position_bytes);
  a->positions = positions;
  a->position_bytes = position_bytes;
  return check_device_range(positions, need * position_bytes, "positions");
}

// Rows (a token of a head) that a workgroup takes about. Few tokens and many heads share
// the angles best, and where the heads are few more tokens make up for them: with 512
// rows, 16 tokens and 32 heads each, prompts of 12,300 tokens and 120 heads were written in 298
// us instead of 247, and with 4 tokens of every kind, prompts of 28 heads over 4 were
// rotated in 84 us instead of 67.
constexpr int64_t kPlaceRows = 128, kFewTokens = 4;

// Eight pairs an item where the head's parts are whole runs of eight.
bool by_eight(const PlaceArgs& a) { return a.head_dim % 16 == 0 && a.pairs % 8 == 0; }

// The workgroups of `tokens` tokens in `spans` spans (0: one after another).
int place_grid(int64_t spans, int64_t tokens, int values, PlaceArgs* a, dim3* grid) {
  int64_t workgroups = 0;
  for (HeadKind& k : a->kinds) {
    k.begin = workgroups;
    k.each = k.groups = k.parts = 1;
    k.chunk = kSpan;
    if (!k.heads) continue;
    int64_t chunk = kFewTokens;
    while (chunk < kSpan && chunk * k.heads < kPlaceRows) chunk *= 2;
    if (k.turned) chunk = std::min<int64_t>(chunk, kMostAngles / a->pairs);
    if (spans) {
      // spans of few tokens, as a decode step's, are not cut
      const bool whole = tokens <= spans * chunk;
      k.parts = whole ? 1 : static_cast<int32_t>(up(kSpan, chunk));
      if (whole) chunk = kSpan;
    } else {
      // fewer tokens where there are few: a thousand workgroups, for 256 CUs
      chunk = std::min(chunk, std::max<int64_t>(1, tokens / 1024));
    }
    const int64_t runs = spans ? spans * k.parts : up(tokens, chunk);
    const int64_t rows = k.heads * std::max<int64_t>(1, std::min(chunk, up(tokens, runs)));
    const int64_t groups = std::max<int64_t>(1, rows / kPlaceRows);
    k.chunk = static_cast<int32_t>(chunk);
    k.each = static_cast<int32_t>(up(k.heads, groups));
    k.groups = static_cast<int32_t>(up(k.heads, k.each));
    workgroups += runs * k.groups;
  }
  a->by_pairs = divisor(std::max(1, a->pairs));
  a->units = divisor(a->head_dim / (2 * values));
  const int rc = check_grid(workgroups, kPlaceLanes);
  *grid = dim3(static_cast<uint32_t>(workgroups));
  return rc;
}

template <typename G, typename T>
int launch_place(PlaceArgs a, int64_t spans, int64_t tokens, hipStream_t stream) {
  constexpr int kValues = sizeof(G) == 4 ? 4 : 8;
  const bool eight = by_eight(a);
  dim3 grid;
  const int rc = place_grid(spans, tokens, eight ? kValues : 1, &a, &grid);
  if (rc || grid.x == 0) return rc;
  return launch(eight ? place_rows_kernel<kValues, G, T> : place_rows_kernel<1, G, T>, grid,
                kPlaceLanes, stream, a, "place_rows_kernel launch");
}

template <typename F>
int by_half_type(int dtype, const F& f) {
  return dtype == AEGKV_DTYPE_BFLOAT16 ? f(__bf16{}) : f(_Float16{});
}

template <typename F>
int by_width(int head_dim, const F& f) {
  switch (head_dim) {
    case 64: return f(Constant<64>{});
    case 128: return f(Constant<128>{});
    default: return f(Constant<256>{});
  }
}

// What one eviction writes belongs to one sequence: the blocks of what stays are
// in no other place of either batch's tables.
int check_targets(const Header& h, const char* host, const Header* into, const char* into_host,
                  int64_t keep) {
  std::vector<uint8_t> use;   // 1: read, 2: written
  try {
    use.resize(static_cast<size_t>(h.num_blocks));
  } catch (const std::exception& e) {
    return fail(AEGKV_ENOMEM, "the tables' blocks: %s", e.what());
  }
  const auto walk = [&](const Header& of, const char* plan, int64_t s, int64_t columns,
                        uint8_t mark) {
    const auto* seq = seqs(plan, of.room) + s;
    const auto* table = reinterpret_cast<const int32_t*>(plan + of.room.at_table) + seq->table;
    for (int64_t c = 0; c < columns; ++c) {
      uint8_t& u = use[static_cast<size_t>(table[c])];
      if (u == 2 || (mark == 2 && u))
        return fail(AEGKV_EDUP, "sequence %lld: block %d is written, and another place of the "
                    "tables has it too", ll(s), table[c]);
      u = mark;
    }
    return 0;
  };
  int rc = 0;
  if (into) {
    for (int64_t s = 0; s < h.num_seqs && !rc; ++s)
      rc = walk(h, host, s, up(seqs(host, h.room)[s].len, h.block_size), 1);
    for (int64_t s = 0; s < h.num_seqs && !rc; ++s)
      rc = walk(*into, into_host, s,
                up(std::min<int64_t>(seqs(host, h.room)[s].len, keep), h.block_size), 2);
    return rc;
  }
  // in place: every block of a sequence that loses tokens is its own alone
  for (int64_t s = 0; s < h.num_seqs && !rc; ++s) {
    const int64_t len = seqs(host, h.room)[s].len;
    rc = walk(h, host, s, up(len, h.block_size), len > keep ? 2 : 1);
  }
  return rc;
}

}  // namespace

extern "C" {

int aegkv_rotate(const aegkv_rotary* rotary, const void* positions, int64_t num_positions,
                 int position_bytes, int32_t head_dim, const aegkv_rows* q, const aegkv_rows* q_out,
                 const aegkv_rows* k, const aegkv_rows* k_out, hipStream_t stream) {
  g_err[0] = '\0';
  if (!rotary || !q || !q_out || !k != !k_out)
    return fail(AEGKV_EINVAL, "rotary, q and what they go to must not be null");
  if (head_dim < 2 || head_dim > 1024 || head_dim % 2)
    return fail(AEGKV_EINVAL, "heads of %d values", head_dim);
  PlaceArgs a = {};
  a.tokens = q->tokens;
  a.head_dim = head_dim;
  if (a.tokens < 0 || a.tokens > kMostTokens)
    return fail(AEGKV_EINVAL, "%lld tokens", ll(a.tokens));
  int rc = check_rotary(rotary, head_dim, &a);
  if (!rc && !positions && a.tokens) rc = fail(AEGKV_EINVAL, "positions must not be null");
  if (!rc) rc = check_positions(positions, num_positions, position_bytes, a.tokens, &a);
  if (rc) return rc;
  const int dtype = q->dtype;
  HeadKind* const kinds[2] = {&a.kinds[0], &a.kinds[1]};
  const aegkv_rows* const from[2] = {q, k};
  const aegkv_rows* const to[2] = {q_out, k_out};
  const char* const names[4] = {"q", "k", "q_out", "k_out"};
  for (int i = 0; i < 2 && from[i] && !rc; ++i) {
    const int32_t heads = from[i]->heads;
    if (heads <= 0 || heads > 65535) return fail(AEGKV_EINVAL, "%s: %d heads", names[i], heads);
    if (from[i]->tokens != a.tokens || to[i]->tokens != a.tokens)
      return fail(AEGKV_EINVAL, "%s: %lld tokens, and %lld to write of %lld", names[i],
                  ll(from[i]->tokens), ll(to[i]->tokens), ll(a.tokens));
    kinds[i]->heads = heads;
    kinds[i]->turned = 1;
    rc = check_rows(from[i], heads, head_dim, dtype, a.tokens, a.tokens, false, false, names[i],
                    &kinds[i]->from);
    if (!rc) rc = check_rows(to[i], heads, head_dim, dtype, a.tokens, a.tokens, false, true,
                             names[2 + i], &kinds[i]->to);
  }
  if (rc || a.tokens == 0) return rc;
  // in place, each item is read by the lane that writes it
  const auto named = [&](int i, bool out) {
    return rows_named(out ? kinds[i]->to : kinds[i]->from, a.tokens, kinds[i]->heads, head_dim,
                      dtype, names[2 * out + i]);
  };
  const Named turns{place(a.turns, int64_t(a.pairs) * 8), "turns"};
  const Named where{place(a.positions, a.tokens * a.position_bytes), "positions"};
  for (int i = 0; i < 2 && from[i] && !rc; ++i) {
    rc = check_apart(named(i, true), {turns, where});
    for (int j = 0; j < 2 && from[j] && !rc; ++j) {
      if (!(i == j && same(named(i, true).at, named(i, false).at)))
        rc = check_apart(named(i, true), {named(j, false)});
      if (i < j && !rc) rc = check_apart(named(i, true), {named(j, true)});
    }
  }
  if (rc) return rc;
  return by_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    return launch_place<T, T>(a, 0, a.tokens, stream);
  });
}

int aegkv_paged_write(const void* plan, const void* device_plan, const aegkv_paged_cache* cache,
                      const aegkv_rows* k, const aegkv_rows* v, const aegkv_rotary* rotary,
                      const void* positions, int64_t num_positions, int position_bytes,
                      const aegkv_rows* q, const aegkv_rows* q_out, hipStream_t stream) {
  PagedCall c;
  int rc = open_paged(plan, device_plan, cache, stream, &c);
  if (rc) return rc;
  const Header& h = c.h;
  const int32_t head_dim = cache->head_dim;
  if (!k || !v) return fail(AEGKV_EINVAL, "k and v must not be null");
  if (!q != !q_out || (q && !rotary) || (positions && !rotary))
    return fail(AEGKV_EINVAL, "q goes to q_out, and only to be rotated, as positions are for");
  PlaceArgs a = {};
  a.plan = c.plan;
  a.at_new_spans = h.room.at_new_spans;
  a.head_dim = head_dim;
  a.page_token = c.pages.token;
  a.page_head = c.pages.head;
  HeadKind &query = a.kinds[0], &key = a.kinds[1], &value = a.kinds[2];
  const int64_t now = h.num_tokens, room = h.room.tokens, tokens = reached(c);
  rc = check_rows(k, h.kv_heads, head_dim, k->dtype, now, room, c.capturing, false, "k",
                  &key.from);
  if (!rc) rc = check_rows(v, h.kv_heads, head_dim, k->dtype, now, room, c.capturing, false, "v",
                           &value.from);
  if (!rc && q) rc = check_rows(q, h.heads, head_dim, cache->dtype, now, room, c.capturing, false,
                                "q", &query.from);
  if (!rc && q) rc = check_rows(q_out, h.heads, head_dim, cache->dtype, now, room, c.capturing,
                                true, "q_out", &query.to);
  if (!rc && rotary) rc = check_rotary(rotary, head_dim, &a);
  if (!rc && positions) rc = check_positions(positions, num_positions, position_bytes, tokens, &a);
  if (rc) return rc;
  query.heads = q ? h.heads : 0;
  key.heads = value.heads = h.kv_heads;
  query.turned = key.turned = rotary != nullptr;
  key.pages = c.pages.k;
  key.block = c.pages.k_block;
  value.pages = c.pages.v;
  value.block = c.pages.v_block;
  const auto rows = [&](const Values& x, int32_t heads, int dtype, const char* what) {
    return rows_named(x, tokens, heads, head_dim, dtype, what);
  };
  const Named kn = rows(key.from, h.kv_heads, k->dtype, "k");
  const Named vn = rows(value.from, h.kv_heads, k->dtype, "v");
  const Named turns{place(a.turns, rotary ? int64_t(a.pairs) * 8 : 0), "turns"};
  const Named where{place(a.positions, positions ? tokens * a.position_bytes : 0), "positions"};
  for (const Named& written : {k_cache(c), v_cache(c)}) {
    rc = check_apart(written, {plan_place(c), kn, vn, turns, where});
    if (rc) return rc;
  }
  rc = check_apart(k_cache(c), {v_cache(c)});
  if (!rc && q) {
    const Named qn = rows(query.from, h.heads, cache->dtype, "q");
    const Named to = rows(query.to, h.heads, cache->dtype, "q_out");
    rc = check_apart(to, {k_cache(c), v_cache(c), plan_place(c), kn, vn, turns, where});
    if (!rc && !same(to.at, qn.at)) rc = check_apart(to, {qn});
    if (!rc) rc = check_apart(qn, {k_cache(c), v_cache(c)});
  }
  if (rc) return rc;
  if (!h.room.new_spans) return 0;
  return by_half_type(cache->dtype, [&](auto t) {
    return by_type(k->dtype, [&](auto given) {
      return launch_place<decltype(given), decltype(t)>(a, h.room.new_spans, room, stream);
    });
  });
}

int aegkv_paged_attend(const void* plan, const void* device_plan, const aegkv_paged_cache* cache,
                       const aegkv_rows* q, const aegkv_rows* out, float* lse, int64_t lse_tokens,
                       int64_t lse_token_stride, double scale, void* workspace,
                       int64_t workspace_bytes, hipStream_t stream) {
  PagedCall c;
  int rc = open_paged(plan, device_plan, cache, stream, &c);
  if (rc) return rc;
  const Header& h = c.h;
  const int32_t head_dim = cache->head_dim;
  const int dtype = cache->dtype;
  PagedAttendArgs a = {};
  float factor;
  rc = check_scale(scale, &factor);
  const int64_t now = h.num_tokens, room = h.room.tokens, tokens = reached(c);
  if (!rc) rc = check_rows(q, h.heads, head_dim, dtype, now, room, c.capturing, false, "q", &a.q);
  if (!rc) rc = check_rows(out, h.heads, head_dim, dtype, now, room, c.capturing, true, "out",
                           &a.out);
  Values sums = {reinterpret_cast<char*>(lse), lse_token_stride, 1, false};
  if (!rc && lse) {
    rc = check_count(lse_tokens, now, room, c.capturing, "lse");
    if (!rc) rc = check_values(lse, lse_tokens, 1, h.heads, AEGKV_DTYPE_FLOAT32, lse_token_stride,
                               h.heads, true, "lse", &sums);
  }
  if (rc) return rc;
  const int64_t floats = parts_floats(h, head_dim, a.kind_work, a.kind_slot_floats);
  if (floats) {
    if (!workspace || !aligned16(workspace) || workspace_bytes < 4 * floats)
      return fail(AEGKV_ENOMEM, "attention over this plan takes a workspace of %lld bytes, "
                  "16-byte aligned", ll(4 * floats));
    rc = check_device_range(workspace, 4 * floats, "the workspace");
    if (rc) return rc;
  }
  const Named from = rows_named(a.q, tokens, h.heads, head_dim, dtype, "q");
  const Named to = rows_named(a.out, tokens, h.heads, head_dim, dtype, "out");
  const Named parts{place(workspace, 4 * floats), "the workspace"};
  const Named log{lse ? rows_place(sums, tokens, 1, h.heads, AEGKV_DTYPE_FLOAT32)
                      : place(nullptr, 0), "lse"};
  // in place every row is read by the workgroup that writes it, or before all that do
  if (!same(from.at, to.at)) rc = check_apart(to, {from});
  if (!rc) rc = check_apart(to, {k_cache(c), v_cache(c), plan_place(c)});
  if (!rc) rc = check_apart(parts, {to, from, k_cache(c), v_cache(c), plan_place(c)});
  if (!rc) rc = check_apart(log, {to, from, parts, k_cache(c), v_cache(c), plan_place(c)});
  if (rc) return rc;
  a.sight = sight_of(h, factor);
  a.pages = c.pages;
  a.plan = c.plan;
  a.at_table = h.room.at_table;
  a.at_merges = h.room.at_merges;
  a.lse = lse;
  a.lse_token = sums.token;
  a.work_base = static_cast<float*>(workspace);
  a.group = h.group;
  rc = check_grid(h.room.merges, 256);
  for (int kind = 0; kind < kKinds && !rc; ++kind)
    rc = check_grid(h.room.items[kind], kPagedLanes);
  if (rc) return rc;
  return by_width(head_dim, [&](auto d) {
    return by_half_type(dtype, [&](auto t) {
      constexpr int kDim = decltype(d)::value;
      typedef decltype(t) T;
      for (int kind = 0; kind < kKinds; ++kind) {
        if (!h.room.items[kind]) continue;
        a.kind = kind;
        a.at_items = h.room.at_items[kind];
        a.work = a.work_base + a.kind_work[kind];
        a.slot_floats = a.kind_slot_floats[kind];
        const auto kernel = kind == kFew    ? paged_attend_kernel<kDim, T, 1>
                            : kind == kMore ? paged_attend_kernel<kDim, T, 2>
                                            : paged_prompt_kernel<kDim, T>;
        const int rc = launch(kernel, dim3(static_cast<uint32_t>(h.room.items[kind])), kPagedLanes,
                              stream, a, "paged_attend_kernel launch");
        if (rc) return rc;
      }
      if (h.room.merges)
        return launch(paged_merge_kernel<kDim, T>, dim3(static_cast<uint32_t>(h.room.merges)), 256,
                      stream, a, "paged_merge_kernel launch");
      return 0;
    });
  });
}

int aegkv_paged_weigh(const void* plan, const void* device_plan, const aegkv_paged_cache* cache,
                      const aegkv_rows* q, const float* lse, int64_t lse_tokens,
                      int64_t lse_token_stride, double scale, float* weights, hipStream_t stream) {
  PagedCall c;
  int rc = open_paged(plan, device_plan, cache, stream, &c);
  if (rc) return rc;
  const Header& h = c.h;
  if (h.shared && !c.capturing)
    return fail(AEGKV_EDUP, "two places of the batch's tables that queries see are one block, "
                "which would gather two sequences' weights at once");
  const int32_t head_dim = cache->head_dim;
  const int dtype = cache->dtype;
  WeighArgs a = {};
  float factor;
  rc = check_scale(scale, &factor);
  const int64_t now = h.num_tokens, room = h.room.tokens, tokens = reached(c);
  if (!rc) rc = check_rows(q, h.heads, head_dim, dtype, now, room, c.capturing, false, "q", &a.q);
  Values sums = {};
  if (!rc) rc = check_count(lse_tokens, now, room, c.capturing, "lse");
  if (!rc) rc = check_values(lse, lse_tokens, 1, h.heads, AEGKV_DTYPE_FLOAT32, lse_token_stride,
                             h.heads, false, "lse", &sums);
  if (rc) return rc;
  const int64_t floats = h.num_blocks * h.kv_heads * h.block_size;
  if (!weights || reinterpret_cast<uintptr_t>(weights) % 4)
    return fail(AEGKV_EINVAL, "weights must not be null, and 4-byte aligned");
  rc = check_device_range(weights, 4 * floats, "weights");
  if (!rc) rc = check_apart(Named{place(weights, 4 * floats), "weights"},
                            {rows_named(a.q, tokens, h.heads, head_dim, dtype, "q"),
                             Named{rows_place(sums, tokens, 1, h.heads, AEGKV_DTYPE_FLOAT32),
                                   "lse"},
                             k_cache(c), v_cache(c), plan_place(c)});
  if (rc) return rc;
  a.sight = sight_of(h, factor);
  a.pages = c.pages;
  a.plan = c.plan;
  a.at_seqs = h.room.at_seqs;
  a.at_table = h.room.at_table;
  a.at_place_tiles = h.room.at_place_tiles;
  a.lse = lse;
  a.lse_token = sums.token;
  a.weights = weights;
  a.group = divisor(h.group);
  a.kv_heads = h.kv_heads;
  // a captured call's batch may hold any tiles that there is room for, under the same rows
  const bool few_rows = h.room.items[kFew] || h.room.items[kMore];
  const int64_t many = !h.room.items[kMany] ? 0 : c.capturing ? h.room.place_tiles : h.many_tiles;
  const int64_t few = !few_rows     ? 0
                      : c.capturing ? h.room.place_tiles
                                    : h.place_tiles - h.many_tiles;
  rc = check_grid(4 * std::max(many, few) * h.kv_heads, kPagedLanes);
  if (rc) return rc;
  const auto grid = [&](int shares, int64_t tiles) {
    return dim3(static_cast<uint32_t>(shares * tiles * h.kv_heads));
  };
  return by_width(head_dim, [&](auto d) {
    return by_half_type(dtype, [&](auto t) {
      constexpr int kDim = decltype(d)::value;
      typedef decltype(t) T;
      int rc = 0;
      if (many)
        rc = launch(paged_weigh_rows_kernel<kDim, T>, grid(kWeighPlaces / kRowsPlaces, many),
                    kPagedLanes, stream, a, "paged_weigh_rows_kernel launch");
      a.first_tile = c.capturing ? 0 : h.many_tiles;
      if (!rc && few)
        rc = launch(paged_weigh_kernel<kDim, T>, grid(4 / weigh_parts(kDim), few), kPagedLanes,
                    stream, a, "paged_weigh_kernel launch");
      return rc;
    });
  });
}

int aegkv_paged_evict(const void* plan, const void* device_plan, const aegkv_paged_cache* cache,
                      float* weights, int64_t keep, int64_t sinks, int64_t recent,
                      const void* into_plan, const void* into_device_plan, int32_t* kept,
                      hipStream_t stream) {
  PagedCall c;
  int rc = open_paged(plan, device_plan, cache, stream, &c);
  if (rc) return rc;
  const Header& h = c.h;
  if (c.capturing)
    return fail(AEGKV_EINVAL, "an eviction is not captured: its batch is another one afterwards");
  if (keep < 1 || keep > kMostTokens || sinks < 0 || recent < 0 || sinks > keep ||
      recent > keep - sinks)
    return fail(AEGKV_EINVAL, "%lld tokens to keep, the first %lld and the last %lld among them",
                ll(keep), ll(sinks), ll(recent));
  if (!h.complete)
    return fail(AEGKV_ERANGE, "some columns of the batch are released: their tokens are gone");
  Header into;
  if (!into_plan != !into_device_plan)
    return fail(AEGKV_EINVAL, "a plan to evict into comes with its device copy");
  if (into_plan) {
    rc = check_plan(into_plan, into_device_plan, &into);
    if (rc) return rc;
    if (into.block_size != h.block_size || into.kv_heads != h.kv_heads ||
        into.num_blocks > cache->num_blocks || into.num_seqs != h.num_seqs || !into.complete)
      return fail(AEGKV_EINVAL, "the plan to evict into is of other sequences or another cache");
    for (int64_t s = 0; s < h.num_seqs; ++s) {
      const int64_t rows = std::min<int64_t>(seqs(plan, h.room)[s].len, keep);
      if (seqs(into_plan, into.room)[s].len < rows)
        return fail(AEGKV_ERANGE, "sequence %lld: %lld tokens into %d places", ll(s), ll(rows),
                    seqs(into_plan, into.room)[s].len);
    }
  }
  Header all = h;    // over the blocks of both plans
  if (into_plan) all.num_blocks = std::max(h.num_blocks, into.num_blocks);
  c.h.num_blocks = all.num_blocks;
  const char* const host = static_cast<const char*>(plan);
  rc = check_targets(all, host, into_plan ? &into : nullptr,
                     static_cast<const char*>(into_plan), keep);
  if (rc) return rc;
  const int64_t count = int64_t(h.num_seqs) * h.kv_heads;
  if (count == 0) return 0;
  const int64_t floats = all.num_blocks * h.kv_heads * h.block_size;
  if (!weights || reinterpret_cast<uintptr_t>(weights) % 4 || !kept ||
      reinterpret_cast<uintptr_t>(kept) % 4)
    return fail(AEGKV_EINVAL, "weights and kept must not be null, and 4-byte aligned");
  if (count > INT64_MAX / 8 / keep) return fail(AEGKV_ERANGE, "kept is larger than any device");
  for (const int64_t bytes : {c.cache.k_block_bytes, c.cache.v_block_bytes})
    if (static_cast<__int128>(all.num_blocks) * bytes > (static_cast<__int128>(1) << 46))
      return fail(AEGKV_ERANGE, "the cache is larger than any device");
  rc = check_device_range(weights, 4 * floats, "weights");
  if (!rc) rc = check_device_range(kept, 4 * count * keep, "kept");
  if (!rc) rc = check_device_range(c.cache.k_pages, (all.num_blocks - 1) * c.cache.k_block_bytes +
                                   c.page_bytes, "the K cache");
  if (!rc) rc = check_device_range(c.cache.v_pages, (all.num_blocks - 1) * c.cache.v_block_bytes +
                                   c.page_bytes, "the V cache");
  const Named w{place(weights, 4 * floats), "weights"};
  const Named to{place(kept, 4 * count * keep), "kept"};
  const Named other{place(into_device_plan, into_plan ? into.room.bytes : 0),
                    "the other plan's device copy"};
  const Named own{place(c.plan, h.room.bytes), "the plan's device copy"};
  if (!rc) rc = check_apart(to, {w, k_cache(c), v_cache(c), own, other});
  if (!rc) rc = check_apart(w, {k_cache(c), v_cache(c), own, other});
  if (!rc) rc = check_apart(k_cache(c), {v_cache(c), own, other});
  if (!rc) rc = check_apart(v_cache(c), {own, other});
  if (rc) return rc;
  EvictArgs a = {};
  a.plan = c.plan;
  a.into_plan = into_plan ? static_cast<const char*>(into_device_plan) : c.plan;
  a.at_seqs = h.room.at_seqs;
  a.at_table = h.room.at_table;
  a.into_at_seqs = into_plan ? into.room.at_seqs : h.room.at_seqs;
  a.into_at_table = into_plan ? into.room.at_table : h.room.at_table;
  a.pages = c.pages;
  a.weights = weights;
  a.kept = kept;
  a.keep = keep;
  a.sinks = sinks;
  a.recent = recent;
  a.kv_heads = h.kv_heads;
  a.block_shift = __builtin_ctz(h.block_size);
  a.row_chunks = cache->head_dim / 8;
  // in place one workgroup takes a sequence's rows in order
  a.rows_each = into_plan ? int64_t(kMoveLanes) / a.row_chunks * kMoveAtOnce : keep;
  int64_t longest = 0;
  for (int64_t s = 0; s < h.num_seqs; ++s)
    longest = std::max<int64_t>(longest, seqs(plan, h.room)[s].len);
  a.groups = static_cast<int32_t>(std::max<int64_t>(1, up(std::min(keep, longest), a.rows_each)));
  const int move_lanes = into_plan ? kMoveLanes : kMostMoveLanes;
  rc = check_grid(count, kSelectLanes);
  if (!rc) rc = check_grid(3 * count * a.groups, move_lanes);
  if (rc) return rc;
  const auto select = longest <= 8 * kSelectLanes    ? paged_select_kernel<8>
                      : longest <= 32 * kSelectLanes ? paged_select_kernel<32>
                                                     : paged_select_kernel<0>;
  rc = launch(select, dim3(static_cast<uint32_t>(count)), kSelectLanes, stream, a,
              "paged_select_kernel launch");
  if (rc) return rc;
  return launch(paged_move_kernel, dim3(static_cast<uint32_t>(3 * count * a.groups)), move_lanes,
                stream, a, "paged_move_kernel launch");
}

}  // extern "C"

#endif  // AEGKV_PAGED_CALLS_H
