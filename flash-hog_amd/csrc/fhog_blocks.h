// Attention over chosen blocks of a paged cache: parameter blocks and the split of its work
// (fhog_block_select.hip, fhog_blocks.hip). A block is a page, named by its column of the page table.
#pragma once

#include "fhog_block_plan.h"
#include "fhog_paged.h"

namespace fhog {

template <typename C> struct KeyMeansParams {
  const C* k;
  const uint8_t* k_scale;
  float* means;  // (pages, kv_heads, head_dim)
  CacheShape at;  // (total: not known, the most)
};

template <typename T> struct BlockSelectParams {
  const T* q;
  const float* means;
  int* chosen;  // (total, kv_heads, blocks)
  CacheShape at;
  unsigned long* scores;  // workspace: (tokens of a slab, kv_heads, pages_per_seq), as sortable bits
  int heads, blocks, first, last;
  int token0, tokens;  // the slab
};

template <typename T, typename C> struct BlockParams {
  const T* q;
  T* out;
  CacheRows<C> cache;
  CacheShape at;
  const int* chosen;
  float* parts;  // as PagedParams'
  int heads, blocks;
  int slots, splits, split_tiles;  // slots: tiles of 16 rows of a token's group, at a time
  int clear_rest;
  float scale;
  int slot0;  // the first of these
};

// How choices are made: by tiles of 16 tokens of a sequence (slots of them), token by token in a workgroup each, or with
// scores in memory, of how many tokens at a time (slab; 0: scores stay in LDS).
struct SelectPlan {
  bool tiles;
  int slots, slab;
};
constexpr long kScoreBytes = 256l << 20;
constexpr int kFusedColumns = 1024;
// Up to kFusedColumns columns: a workgroup a token and head, up to 512 of them; a tile's workgroup reads the means once for
// 16 tokens, but chooses for them four at a time; with scores in memory every token reads the means and another launch
// chooses. us, tiles / tokens / memory, 250 columns of D128: 1 token of 8 heads 13 / 10 / 12, 64 tokens of one sequence
// 30 / 14 / 14, 16 sequences of 4 14 / 14 / 14, 64 of 2 24 / 25 / 20, 256 of 1 52 / 47 / 35, 64 of 4 25 / 42 / 35, 64 of 8
// 27 / 75 / 66; 1000 columns: 41 / 23 / 20, 80 / 35 / 40, 43 / 37 / 43, 86 / 69 / 74; 1000 of D256, 2 heads, where a token's
// workgroup would wait for 1 MB by itself: 63 / 73 / 19, 102 / 76 / 28, 66 / 81 / 39, 67 / 104 / 59.
// Wider tables have no kernel of their own, scores go through memory and, in up to nine passes, back: with 1026 / 1027 / 2048 / 8192
// columns 2048 tokens of 8 heads of 128 take 175 / 208 / 389 / 1675 us, 16 single tokens 18 / 25 / 37 / 164, one of 4 heads of 64
// 12 / 13 / 18 / 52.
inline SelectPlan select_plan(int batch, int total, bool single, int kv_heads, int head_dim, int pages_per_seq, int first, int last) {
  SelectPlan p;
  p.slots = total / 16 + batch;
  long fit = kScoreBytes / (8l * kv_heads * pages_per_seq);
  if (fit > (1l << 22) / kv_heads) fit = (1l << 22) / kv_heads;  // (a launch's threads are 32 bits)
  p.slab = (int)(fit < 1 ? 1 : fit < total ? fit : total);
  const long columns = (long)pages_per_seq - first - last, rows = (long)total * kv_heads;
  if (columns > kFusedColumns) {
    p.tiles = !single && total >= 8l * batch;
    return p;
  }
  p.tiles = false;
  if (head_dim <= 128 && rows <= 512) {
    p.slab = 0;
    return p;
  }
  const double n = columns > 0 ? (double)columns : 0.;
  const int each = total < 16l * batch ? (total + batch - 1) / batch : 16, held = n <= 256 ? 1024 : n <= 512 ? 512 : 256;
  const double full = (double)p.slots * kv_heads / held;  // of the tiles that 256 CUs hold
  const double tile_us = (full < 1 ? 1 : full) * (4 + n * head_dim * 1.9e-4 + (each + 3) / 4 * (2.5 + 0.0105 * n));
  const double memory_us = 10 + rows * n * head_dim * 4 / 5.5e6;
  if (!single && tile_us < memory_us) {
    p.tiles = true;
    p.slab = 0;
  }
  return p;
}

// Attention of tokens over chosen blocks: tiles of 16 rows, and how the blocks are split.
struct BlockPlan {
  int slots, splits, split_tiles;
  int slab;    // slots at a time: as many as leave no more than kPartBytes of parts
  long parts;  // rows of them
};
constexpr int kSplitBlocks = 512;  // blocks of a split, whose places are in LDS
inline BlockPlan block_plan(int total, int heads, int kv_heads, int head_dim, int page_size, int blocks, int cus) {
  if (cus <= 0) cus = 256;
  BlockPlan p;
  p.slots = total * ((heads / kv_heads + 15) / 16);
  const long tiles = ((long)blocks * page_size + 31) / 32;
  const int waves = head_dim == 64 ? 8 : head_dim == 128 ? 4 : 2;
  // Few long splits: a workgroup's start, four dependent loads, is as long as its walk over 500 keys. (Eight / four / two /
  // one a CU, us, without the join, which one split does without: B16 x 64 blocks of 64, H32/8 D128 e4m3 38 / 30 / 26 / 27,
  // B32 x 32 of 32 bf16 34 / 28 / 25 / 25, B64 x 64 of 16, H16/4 D64 18 / 18 / 15 / 15, B8 x 32 of 64 e4m3 17 / 17 / 13 / 12.)
  const long work = (long)p.slots * kv_heads;
  long splits = work >= cus ? 1 : (cus + work - 1) / work;
  if (splits > tiles / waves) splits = tiles / waves;
  // (the join costs 3 us: up to four tiles a wave go without. B1 x 32 of 16, H16/4 D64 7.0, in two splits 9.2; B16 x 32 of 32,
  // H12/12 D64 12.4, in two 16.5; B1 x 16 of 64, H32/8 D128, eight tiles a wave, 9.8 in eight splits, in two 13.6)
  if (tiles <= 4l * waves) splits = 1;
  if (splits > kJoinWeights / 16) splits = kJoinWeights / 16;
  const long needed = (tiles * 32 + (long)(kSplitBlocks - 1) * page_size - 1) / ((long)(kSplitBlocks - 1) * page_size);
  if (splits < needed) splits = needed;
  if (splits < 1) splits = 1;
  p.split_tiles = (int)((tiles + splits - 1) / splits);
  p.splits = (int)((tiles + p.split_tiles - 1) / p.split_tiles);
  // (lists of more than kSplitBlocks have several splits however many tokens there are)
  const long rows = p.splits > 1 ? (long)kv_heads * p.splits * 16 : 0, fit = rows ? kPartBytes / (rows * (head_dim + 2) * 4) : p.slots;
  p.slab = (int)(fit < 1 ? 1 : fit < p.slots ? fit : p.slots);
  p.parts = p.slab * rows;
  return p;
}

// Attention of many tokens, a block at a time (fhog_blocks_chunk.hip, fhog_block_plan.h).
struct PackedTokenAt {
  int pos;  // -1: of no sequence
};
template <typename T, typename C> struct BlockChunkParams {
  const T* q;
  T* out;
  CacheRows<C> cache;
  CacheShape at;
  const int* chosen;
  int heads, blocks, clear_rest;
  float scale;
  int lists;           // batch * kv_heads * pages_per_seq
  int token0, tokens;  // the slab
  int groups;          // of 64 of its tokens
  // workspace
  unsigned long* masks;     // (kv_heads, groups, pages_per_seq) which of a group's tokens chose each column
  unsigned long* falling;   // (kv_heads, groups) whose lists do not rise
  int* before;              // (kv_heads, groups, pages_per_seq) entries of a list before the group
  int* base;                // (lists) its first tile
  BlockEntryAt* entries;    // (items, kTileRows)
  BlockItem* items;
  int* total;               // of them; whether the offsets fall somewhere
  float* parts;      // (tokens, kv_heads, blocks, group, head_dim)
  float* parts_ml;   // and their maxima and sums
};
// Lays the workspace (16-byte aligned) out, larger elements first.
template <typename T, typename C> void block_chunk_workspace(BlockChunkParams<T, C>& p, const BlockChunkPlan& plan, int head_dim, void* ws) {
  p.items = (BlockItem*)ws;
  p.parts = (float*)(p.items + plan.items);
  p.parts_ml = p.parts + plan.parts * head_dim;
  p.entries = (BlockEntryAt*)(p.parts_ml + plan.parts * 2);
  p.masks = (unsigned long*)(p.entries + plan.entries);
  p.falling = p.masks + plan.masks;
  p.before = (int*)(p.falling + plan.groups);
  p.base = p.before + plan.masks;
  p.total = p.base + plan.lists;
}
template <typename T, typename C, int D>
hipError_t launch_block_chunk(const BlockChunkParams<T, C>& p, int slab, hipStream_t s);
template <typename C, int D> hipError_t launch_key_means(const KeyMeansParams<C>& p, int workgroups, hipStream_t s);
template <typename T, int D> hipError_t launch_block_select(const BlockSelectParams<T>& p, SelectPlan plan, hipStream_t s);
template <typename T, typename C, int D> hipError_t launch_block_attention(const BlockParams<T, C>& p, int slab, hipStream_t s);

}  // namespace fhog
