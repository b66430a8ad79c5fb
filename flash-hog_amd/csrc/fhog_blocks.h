// Attention over chosen blocks of a paged cache: parameter blocks and the split of its work
// (fhog_block_select.hip, fhog_blocks.hip). A block is a page, named by its column of the page table.
#pragma once

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
  double* scores;  // workspace: (tokens of a slab, kv_heads, pages_per_seq)
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
  int slots, splits, split_tiles;  // slots: tiles of 16 rows of a token's group
  int clear_rest;
  float scale;
};

// A token's scores, of all columns and key/value heads, are 8 bytes each; tokens are taken in slabs that keep
// them within this.
constexpr long kScoreBytes = 256l << 20;
inline int select_slab(int total, int kv_heads, int pages_per_seq) {
  long fit = kScoreBytes / (8l * kv_heads * pages_per_seq);
  if (fit > (1l << 22) / kv_heads) fit = (1l << 22) / kv_heads;  // (a launch's threads are 32 bits)
  return (int)(fit < 1 ? 1 : fit < total ? fit : total);
}

// Attention of tokens over chosen blocks: tiles of 16 rows, and how the blocks are split.
struct BlockPlan {
  int slots, splits, split_tiles;
  long parts;
};
constexpr int kSplitBlocks = 512;  // blocks of a split, whose places are in LDS
inline BlockPlan block_plan(int total, int heads, int kv_heads, int head_dim, int page_size, int blocks, int cus) {
  if (cus <= 0) cus = 256;
  BlockPlan p;
  p.slots = total * ((heads / kv_heads + 15) / 16);
  const long tiles = ((long)blocks * page_size + 31) / 32;
  const int waves = head_dim == 64 ? 8 : head_dim == 128 ? 4 : 2;
  const long work = (long)p.slots * kv_heads, target = 8l * cus;
  long splits = work >= target ? 1 : (target + work - 1) / work;
  const long least = work < 2l * cus ? waves : 4l * waves;
  if (splits > tiles / least) splits = tiles / least;
  if (splits > kJoinWeights / 16) splits = kJoinWeights / 16;
  const long needed = (tiles * 32 + (long)(kSplitBlocks - 1) * page_size - 1) / ((long)(kSplitBlocks - 1) * page_size);
  if (splits < needed) splits = needed;
  if (splits < 1) splits = 1;
  p.split_tiles = (int)((tiles + splits - 1) / splits);
  p.splits = (int)((tiles + p.split_tiles - 1) / p.split_tiles);
  p.parts = p.splits > 1 ? work * p.splits * 16 : 0;
  return p;
}

template <typename C, int D> hipError_t launch_key_means(const KeyMeansParams<C>& p, int workgroups, hipStream_t s);
template <typename T, int D> hipError_t launch_block_select(const BlockSelectParams<T>& p, hipStream_t s);
template <typename T, typename C, int D> hipError_t launch_block_attention(const BlockParams<T, C>& p, hipStream_t s);

}  // namespace fhog
