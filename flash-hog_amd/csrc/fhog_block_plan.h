// Attention of many tokens over chosen blocks, a block at a time (fhog_blocks_chunk.hip): when it is taken, its slabs,
// its workspace, and what of its arrays a workgroup reads. Plain C++.
#pragma once

#include <cstddef>

namespace fhog {

constexpr int kTileRows = 128;       // rows of a tile
constexpr int kMostColumns = 8192;   // of the page table (the masks of 64 tokens are in LDS, 64 KB)
constexpr int kSumBlocks = 256;      // blocks of a list (a join's weights are)
// Sequences times heads times columns: each of their lists adds an item and 128 entries to the workspace, 1 KB. A bound on
// memory, not where the two ways cross: us a token / a block at a time, bf16 H32/8 D128, 16 blocks of 64, one list too many for it:
// 4 sequences of 512 tokens, 1025 columns, at 8192 keys 555 / 264, at 65536 857 / 505; 32 of 64, 129 columns 587 / 502; 16 of
// 128, 1024 columns 571 / 406; 64 of 32, 256 columns 640 / 795; 16 of 512 of H8/8, 1025 columns 2049 / 424.
constexpr int kMostLists = 32768;
// A tile of a list (the tokens that chose one column of a sequence, for one head): whole tokens, whose entries are
// the tile's own kTileRows.
struct BlockItem {
  int rows;
  int page, hk;
  int key0;   // the column's first position
  int shift;  // positions above the tokens' indexes in the slab
  int pad[3];
};
constexpr int tile_tokens(int group) { return kTileRows / group; }
struct BlockEntryAt {
  int token, slot;  // of the slab; where its list has the column, first of all
};

// Indexes [begin, end).
struct IndexRange {
  int begin, end;
};
// Which of a slab's tokens are the packed rows [begin, end), as indexes from its first on. All of a sequence's rows may lie
// before the slab or behind it: both ends are cut to [0, tokens], so that no index of a group of 64 leaves the slab's groups.
constexpr IndexRange slab_range(int begin, int end, int token0, int tokens) {
  begin = begin < token0 ? 0 : begin - token0 < tokens ? begin - token0 : tokens;
  end = end < token0 ? 0 : end - token0 < tokens ? end - token0 : tokens;
  return {begin, end < begin ? begin : end};
}
// The groups of 64 that have some of these tokens: part `way` of `ways` of them.
constexpr IndexRange list_groups(IndexRange of, int way, int ways) {
  if (of.begin >= of.end) return {0, 0};
  const int first = of.begin / 64, last = (of.end + 63) / 64, each = (last - first + ways - 1) / ways;
  const int begin = first + way * each < last ? first + way * each : last;
  return {begin, begin + each < last ? begin + each : last};
}

// Tokens are taken in slabs whose outputs and masks stay within this: each slab has five launches, and ends with CUs idle
// (540 MB of outputs in slabs of 256 / 512 / 1024 MB: 415 / 429 / 394 us; in slabs of 256 / 512 / 1024 / 2048 MB: 4096 tokens of
// H32/8 D128, 1.1 GB, 600 / 499 / 475 / 458, 16384 tokens, 4.4 GB, 2439 / 1968 / 1893 / 1911). Where the outputs would not stay
// in the cache behind the L2s, they are stored past it: tiles / sum of 540 MB 189 / 105 us in it, 134 / 107 past it; of
// 207 MB 60 / 51 and 59 / 59.
constexpr long kPartBytes = 1l << 30, kCacheBytes = 256l << 20;
// Outputs, and masks with the counts before them, of 64 tokens.
inline long block_group_bytes(int heads, int kv_heads, int head_dim, int pages_per_seq, int blocks) {
  return 64l * heads * blocks * (head_dim + 2) * 4 + kv_heads * (12l * pages_per_seq + 8);
}
struct BlockChunkPlan {
  int slab;
  long lists, masks, groups, entries, items, parts;  // elements
  size_t bytes;
};
inline BlockChunkPlan block_chunk_plan(int batch, int total, int heads, int kv_heads, int head_dim, int pages_per_seq, int blocks) {
  BlockChunkPlan p;
  // (64 at least: block_chunk_rule)
  const long fit = kPartBytes / block_group_bytes(heads, kv_heads, head_dim, pages_per_seq, blocks) * 64;
  p.slab = (int)(fit < total ? fit : total);
  p.lists = (long)batch * kv_heads * pages_per_seq;
  p.groups = (long)kv_heads * ((p.slab + 63) / 64);
  p.masks = p.groups * pages_per_seq;
  p.items = (long)p.slab * blocks * kv_heads / tile_tokens(heads / kv_heads) + p.lists;
  p.entries = p.items * kTileRows;
  p.parts = (long)p.slab * heads * blocks;
  p.bytes = (size_t)(p.parts * (head_dim + 2) * 4 + p.items * sizeof(BlockItem) + p.entries * sizeof(BlockEntryAt) +
                     (p.masks + p.groups) * 8 + (p.masks + p.lists + 2) * 4);
  return p;
}
// Whether a call goes a block at a time: where its estimate is below that of a token at a time. A chosen block of a token
// and head (an entry) costs a token's kernel its keys and values out of a cache, at 14 TB/s with 16-bit elements; a block at
// a time costs it fp32 outputs written and read, at 3.8 TB/s both ways, and each listed block its keys and values once. Five
// more launches are 16 us. (us a block / a token at a time, table of 8192 positions, bf16: H32/8 D128, 16 blocks of 64, one
// sequence of 8 / 32 / 128 / 512 / 2048 tokens 24 / 12, 30 / 17, 45 / 42, 79 / 145, 250 / 543; 16 sequences of 2 / 8 / 32 tokens
// 47 / 20, 57 / 43, 92 / 145. One of 2048 tokens: H8/8 83 / 500, H32/4 256 / 306, H8/1 D256 195 / 172, blocks of 32 246 / 353;
// of 512, 32 blocks of 16 166 / 91. e4m3 takes a token's kernel 8 to 25 % less; the sides change where they are as near.)
inline bool block_chunk_rule(int batch, int total, int heads, int kv_heads, int head_dim, int page_size, int pages_per_seq,
                             int blocks, bool single) {
  const int group = heads / kv_heads;
  const long lists = (long)batch * kv_heads * pages_per_seq;
  if (single || pages_per_seq > kMostColumns || blocks > kSumBlocks || group > kTileRows || lists > kMostLists ||
      block_group_bytes(heads, kv_heads, head_dim, pages_per_seq, blocks) > kPartBytes)
    return false;
  const double entries = (double)total * kv_heads * blocks, block = 4.0 * page_size * head_dim;
  const double token_us = entries * block / 14e6;
  const double block_us = 16 + entries * 8.0 * group * (head_dim + 2) / 3.8e6 + (entries < lists ? entries : lists) * block / 14e6;
  return block_us < token_us;
}

}  // namespace fhog
