// The plan of one batch over a quantised paged cache: what aegkv_batch_plan
// lays out in a caller's buffer (plan.cpp) and the kernels of quant_cache.h
// read from its copy on the device. Internal to the library.
#ifndef AEGKV_BATCH_PLAN_H
#define AEGKV_BATCH_PLAN_H

#include <cstdint>

namespace aegkv_batch {

constexpr uint64_t kMagic = 0x314e414c50425141ull;

// Tokens are written and read in spans of 16 (a span lies in one block) and
// attended over in tiles of 32.
constexpr int kSpan = 16;
constexpr int kTile = 32;

// Row r of a sequence's queries under one KV head is new token r / group,
// query head kv_head * group + r % group. Attention takes rows by kind:
//   kFew, kMore: up to 16 rows of a sequence, or up to 64 in blocks of 32; the
//                four waves of a workgroup take an item's tiles in turn and
//                join at its end;
//   kMany:       blocks of kManyRows rows, shared out to the waves.
// 64 sequences of 2,000 tokens, 8 KV heads: 20, 40 and 64 rows take 37, 68 and 70 us as
// kMore, 75, 85 and 87 as kMany; 128 rows 127 and 101.
enum Kind { kFew = 0, kMore = 1, kMany = 2, kKinds = 3 };
constexpr int kManyRows = 128;
constexpr int kKindRows[kKinds] = {16, 32, kManyRows};
constexpr int64_t kMostMore = 64;   // rows of a sequence

struct Seq {
  int32_t len;         // positions in the cache, the new ones included
  int32_t fresh;       // new tokens: positions len - fresh .. len - 1
  int32_t table;       // first entry of its block table
  int32_t token;       // row of its first new token
  int32_t read_span;   // spans of all tokens before this sequence
  int32_t pad;
  int64_t read_token;  // tokens before this sequence
};
static_assert(sizeof(Seq) == 32, "Seq layout");

// Up to 16 new tokens of a sequence inside one block.
struct NewSpan {
  int32_t block, inside, count;
  int32_t token;       // row of the first
};
static_assert(sizeof(NewSpan) == 16, "NewSpan layout");

// One workgroup's work: rows [row, row + rows) of a sequence under one KV head over visited tiles
// [tile, tile_end). Visited tile v is the cache's tile v below `first_tiles` (the
// first tokens that stay visible), else v - first_tiles + window_tile.
struct Item {
  int32_t seq, kv_head, row, rows;
  int32_t tile, tile_end, first_tiles, window_tile;
  int32_t slot;        // where its part of the sum goes; -1: it is the whole
  int32_t base, token, table;   // the sequence's first new position, token row, table
};
static_assert(sizeof(Item) == 48, "Item layout");

// Rows whose tiles were cut into `parts` items with consecutive slots, as one
// workgroup joins them: up to kMergeRows rows of up to as many parts, or one row.
// Row i of them is row `row` + i of the sequence and `first` + i of the items.
constexpr int kMergeRows = 8;
struct Merge {
  int32_t seq, kv_head, row, rows;
  int32_t slot, parts, kind, token;
  int32_t first, pad[3];
};
static_assert(sizeof(Merge) == 48, "Merge layout");

// What a plan has room for; fixed when it is made. Offsets into the buffer
// follow from it, so that a captured launch stays right across updates.
struct Room {
  int64_t bytes;
  int64_t seqs, columns, tokens;   // sequences, table entries, new tokens
  int64_t new_spans, read_spans;
  int64_t items[kKinds];           // a workgroup each; 0: no such kernel is launched
  int64_t slots[kKinds];
  int64_t merges;
  int64_t at_seqs, at_table, at_new_spans, at_items[kKinds], at_merges;
};

struct Header {
  uint64_t magic;
  Room room;
  int64_t num_blocks;
  int32_t block_size, kv_heads, heads, group;
  int32_t window, sinks;           // window 0: none
  int32_t num_seqs, num_tokens;
  int32_t new_spans, read_spans;
  int32_t items[kKinds], slots[kKinds];
  int32_t merges;
  int32_t complete;                // every position of every sequence has its block
  int64_t read_tokens;
};

inline const Seq* seqs(const void* p, const Room& r) {
  return reinterpret_cast<const Seq*>(static_cast<const char*>(p) + r.at_seqs);
}

}  // namespace aegkv_batch

#endif  // AEGKV_BATCH_PLAN_H
