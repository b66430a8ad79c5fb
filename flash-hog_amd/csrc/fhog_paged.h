// The paged key/value cache: parameter blocks, launch rules and the device code that its
// kernels share.
//
// A cache is (pages, kv_heads, page_size, head_dim): the rows of one head in a page are
// contiguous, so a workgroup that serves one key/value head reads whole lines. Page sizes
// are powers of two from 16 on, so that 16 keys from a multiple of 16 on never leave a page.
// Token s of sequence b is row s % page_size of page table[b][s / page_size].
//
// The new tokens of all sequences are packed: sequence b's are rows offsets[b] to
// offsets[b + 1], or row b alone without offsets, and its last `rows` positions: token i
// of its n new ones is at position lengths[b] - n + i.
//
// Nothing on the device is trusted: a table entry outside [0, pages) or a length beyond the
// table's capacity gives NaN in rows of its sequence (attention, reading) or is
// skipped (writing); offsets are cut to [0, total]. No access leaves its tensor.
//
// An e4m3 cache has an e8m0 scale for each key and value row, (pages, kv_heads, page_size):
// the row's values are code * 2^(scale byte - 127).
#pragma once

#include "fhog_device.h"

namespace fhog {

struct e4m3 {  // one byte of an e4m3 cache
  uint8_t byte;
};

struct CacheShape {
  const int* table;    // (batch, pages_per_seq)
  const int* lengths;  // (batch)
  const int* offsets;  // (batch + 1), or null: one new token each
  int batch, total;    // sequences, packed rows
  int kv_heads, pages, page_shift, pages_per_seq;
};

template <typename C> struct CacheRows {
  const C* k;
  const C* v;
  const uint8_t* k_scale;  // e4m3 only
  const uint8_t* v_scale;
};

template <typename T, typename C> struct PagedParams {
  const T* q;
  T* out;
  CacheRows<C> cache;
  CacheShape at;
  float* parts;  // fp32 outputs of the splits, (slot, kv_head, split, row of the tile, head_dim), and their m, l
  int heads, window, sinks;  // window 0: none
  int slots, splits, split_tiles;
  int longest_first;  // PagedPlan
  int clear_rest;  // whether rows of no sequence are zeroed
  float scale;
};

template <typename T, typename C> struct CacheWriteParams {
  const T* k;
  const T* v;
  C* k_cache;
  C* v_cache;
  uint8_t* k_scale;
  uint8_t* v_scale;
  CacheShape at;
};

template <typename T, typename C> struct CacheReadParams {
  CacheRows<C> cache;
  T* k;
  T* v;
  CacheShape at;
  int max_length;
};

template <typename T, typename C, int D> hipError_t launch_paged_attention(const PagedParams<T, C>& p, int rows, hipStream_t s);
template <typename T, typename C, int D> hipError_t launch_cache_write(const CacheWriteParams<T, C>& p, hipStream_t s);
template <typename T, typename C, int D> hipError_t launch_cache_read(const CacheReadParams<T, C>& p, hipStream_t s);

// ---------------------------------------------------------------------------
// Packed rows and their sequences.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int packed_begin(const CacheShape& c, int b) {
  return c.offsets ? min(max(c.offsets[b], 0), c.total) : b;
}

// The last sequence whose first slot is at or before `slot`, where a sequence's slots start
// at offset * group / tile + index (PagedPlan); any answer in range if offsets do not rise.
template <typename F> __device__ __forceinline__ int last_at_or_before(int count, int slot, F&& first_slot) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_slot(mid) <= slot)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A wave's sum over its lanes, in every lane.
__device__ __forceinline__ int wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return __builtin_amdgcn_readlane(x, 63);
}

// A lane's sum over the lanes before it, and in `total` the wave's.
__device__ __forceinline__ int wave_scan(int x, int& total) {
  const int lane = threadIdx.x & 63;
  int through = x;
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(through, d, 64);
    if (lane >= d) through += y;
  }
  total = __shfl(through, 63, 64);
  return through - x;
}

// The same over the threads of a workgroup of THREADS; box: an int a wave, in LDS.
template <int THREADS> __device__ __forceinline__ int group_scan(int x, int& total, int* box) {
  const int wave = threadIdx.x >> 6;
  int sum;
  const int before = wave_scan(x, sum);
  __syncthreads();  // (the box's last use)
  if ((threadIdx.x & 63) == 0) box[wave] = sum;
  __syncthreads();
  int more = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) more += box[w];
    total += box[w];
  }
  return before + more;
}

// Sequence and tile (of ROWS rows) that come at place `order` when all tiles are sorted by the keys
// that their last rows see, most first, then by sequence: at most 64 sequences, one a lane. False
// behind the last tile.
template <int ROWS>
__device__ __forceinline__ bool longest_first(const CacheShape& c, int group, int order, int lane, int& seq, int& tile) {
  const bool mine = lane < c.batch;
  const int begin = mine ? packed_begin(c, lane) : 0;
  const int count = mine ? max(0, packed_begin(c, lane + 1) - begin) : 0;
  const int before = mine ? min(max(0, c.lengths[lane]), 1 << 30) - count : 0;  // keys before the new ones
  const long rows = (long)count * group;
  const int tiles = (int)((rows + ROWS - 1) / ROWS);
  // How many of this lane's tiles see at least `keys` keys: those from the tile of the first row that does.
  auto at_least = [&](int keys) {
    const long row = max(0l, ((long)keys - 1 - before) * group);
    return row < rows ? tiles - (int)(row / ROWS) : 0;
  };
  if (order >= wave_sum(tiles)) return false;
  int lo = count > 0 ? before : 0x7fffffff, hi = count > 0 ? before + count : -0x7fffffff;
  for (int d = 1; d < 64; d <<= 1) {
    lo = min(lo, __shfl_xor(lo, d, 64));
    hi = max(hi, __shfl_xor(hi, d, 64));
  }
  // The most keys that more than `order` tiles see: all see lo, none more than hi.
  hi = __builtin_amdgcn_readfirstlane(hi) + 1;
  lo = __builtin_amdgcn_readfirstlane(lo);
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (wave_sum(at_least(mid)) > order)
      lo = mid;
    else
      hi = mid;
  }
  // Among the tiles that see exactly lo, in order of their lanes.
  const int more = at_least(lo + 1), equal = at_least(lo) - more;
  int through = equal;
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(through, d, 64);
    if (lane >= d) through += x;
  }
  const int place = order - wave_sum(more) - (through - equal);
  const unsigned long here = __ballot(place >= 0 && place < equal);
  seq = __builtin_amdgcn_readfirstlane(here ? __builtin_ctzl(here) : 0);
  tile = __builtin_amdgcn_readlane(tiles - 1 - more - place, seq);
  return here != 0;
}

// ---------------------------------------------------------------------------
// Tiles of cached rows: fetched from their pages into registers, 16 bytes of cache a thread
// and load, and stored to LDS as T, swizzled, where the matrix operands are read. e4m3 rows
// are scaled in between; the scale is a power of two, so bf16 holds the product exactly and
// fp16 wherever its range does.
// ---------------------------------------------------------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Four e4m3 values (the bytes of x) times a power of two, as T.
template <typename T> __device__ __forceinline__ V4<T> dequantise4(uint32_t x, float scale) {
  u32x2 y;
  if constexpr (std::is_same_v<T, __bf16>) {
    y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false));
    y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true));
  } else {
    y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, false));
    y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, true));
  }
  return __builtin_bit_cast(V4<T>, y);
}
// The power of two that an e8m0 code stands for.
__device__ __forceinline__ float scale_of(uint32_t code) { return __builtin_bit_cast(float, code << 23); }

// Where a tile's two halves of 16 keys lie: the line (row of a head of a page) of each half's first key, and
// the last of its rows that is read (the others repeat it, so that what no token has written is never read).
struct HalfRows {
  long line[2];
  int last[2];
  __device__ __forceinline__ long of(int row) const {
    return (row < 16 ? line[0] : line[1]) + min(row & 15, row < 16 ? last[0] : last[1]);
  }
};

// TENSORS: 2 for keys and values, 1 for values alone.
template <typename T, typename C, int D, int THREADS, int SWZ, int TENSORS = 2> struct PageTile {
  static constexpr bool kQuantised = sizeof(C) == 1;
  static constexpr int kPerLoad = 16 / (int)sizeof(C);  // elements
  static constexpr int kChunks = D / kPerLoad;          // 16-byte pieces of a row
  static constexpr int kTensor = 32 * kChunks;          // of a tile of one tensor
  static constexpr int kLoads = TENSORS * kTensor / THREADS;  // a thread's
  static constexpr int kTileBytes = 32 * D * (int)sizeof(T);
  static_assert(TENSORS * kTensor % THREADS == 0, "tile must divide into whole loads");
  u32x4 data[kLoads];
  uint32_t code[kQuantised ? kLoads : 1];

  // Rows [rlo, rhi] of the 32 keys from k0 (a multiple of 16) on; rows outside repeat the
  // nearest of them, so that what no token has written is never read. page[h] is the
  // page of keys k0 + 16 h and on.
  __device__ __forceinline__ void fetch(const CacheRows<C>& cache, int hk, int kv_heads, int page_shift, int k0,
                                        int rlo, int rhi, int page0, int page1, int thread) {
    const int page_rows = 1 << page_shift;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * THREADS + thread;
      const bool value = TENSORS == 1 || at >= kTensor;
      const int row = min(max(at % kTensor / kChunks, rlo), rhi);
      const long head = (long)(row < 16 ? page0 : page1) * kv_heads + hk;
      const long line = (head << page_shift) + ((k0 + row) & (page_rows - 1));
      const C* src = (value ? cache.v : cache.k) + line * D + at % kChunks * kPerLoad;
      data[i] = *reinterpret_cast<const u32x4*>(src);
      if constexpr (kQuantised) code[i] = (value ? cache.v_scale : cache.k_scale)[line];
    }
  }

  __device__ __forceinline__ void fetch(const CacheRows<C>& cache, const HalfRows& rows, int thread) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * THREADS + thread;
      const bool value = TENSORS == 1 || at >= kTensor;
      const long line = rows.of(at % kTensor / kChunks);
      const C* src = (value ? cache.v : cache.k) + line * D + at % kChunks * kPerLoad;
      data[i] = *reinterpret_cast<const u32x4*>(src);
      if constexpr (kQuantised) code[i] = (value ? cache.v_scale : cache.k_scale)[line];
    }
  }

  // To LDS: the tile of keys at byte address lds, that of values behind it (or there).
  __device__ __forceinline__ void store(uint32_t lds, int thread) const {
    typedef __attribute__((address_space(3))) char lds_char;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * THREADS + thread;
      const int row = at % kTensor / kChunks, chunk = at % kChunks;
      const uint32_t base = lds + (TENSORS == 2 && at >= kTensor ? kTileBytes : 0) + row * D * (int)sizeof(T);
      auto put = [&](int c, u32x4 x) {
        *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(
            reinterpret_cast<lds_char*>((uintptr_t)(base + 16 * phys_chunk<SWZ>(row, c)))) = x;
      };
      if constexpr (kQuantised) {
        const float scale = scale_of(code[i]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const V4<T> a = dequantise4<T>(data[i][2 * h], scale), b = dequantise4<T>(data[i][2 * h + 1], scale);
          put(2 * chunk + h, __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)));
        }
      } else {
        put(chunk, data[i]);
      }
    }
  }
};

// PageTile's rows straight to LDS, for 2-byte caches: each load a wave's LDS DMA from one half of the
// tile, whose rows lie in one page, so that the address is the half's first row, uniform, and a
// lane's offset from it, the same for every whole tile.
template <typename T, int D, int THREADS, int SWZ> struct PageDma {
  static constexpr int kRowBytes = D * (int)sizeof(T);
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kWaveRows = 64 / kChunks;               // of a load
  static constexpr int kEach = 32 * kChunks / THREADS;         // a wave's loads of one tensor
  static constexpr int kLoads = 2 * kEach;
  static constexpr int kTileBytes = 32 * kRowBytes;
  static_assert(32 * kChunks % THREADS == 0 && 16 % kWaveRows == 0, "tile must divide into whole loads of a half");
  int wave, lane;
  uint32_t voff[kEach];

  __device__ __forceinline__ int first_row(int i) const { return i * (THREADS / kChunks) + wave * kWaveRows; }
  __device__ __forceinline__ uint32_t chunk(int i) const {
    return 16u * (uint32_t)phys_chunk<SWZ>(first_row(i) + lane / kChunks, lane % kChunks);
  }
  // wave (uniform) and lane within the THREADS threads that fill a tile.
  __device__ __forceinline__ PageDma(int wave_, int lane_) : wave(wave_), lane(lane_) {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      voff[i] = (uint32_t)((first_row(i) & 15) + lane / kChunks) * kRowBytes + chunk(i);
  }
  // Where a tile's halves begin: the byte offset of the first row of each that is read. In their
  // lowest bits, which rows leave free: whether a page is none (the first's), and whether rows
  // of the tile are not read (the second's).
  struct Place {
    long half[2];
  };
  __device__ __forceinline__ static Place place(const CacheShape& c, int hk, int k0, int rlo, int rhi, int page0,
                                                int page1) {
    const bool none = (unsigned)page0 >= (unsigned)c.pages || (unsigned)page1 >= (unsigned)c.pages;
    if (none) page0 = page1 = 0;
    const int in_page = (1 << c.page_shift) - 1;
    auto row = [&](int page, int r) {
      return ((((long)page * c.kv_heads + hk) << c.page_shift) + ((k0 + r) & in_page)) * kRowBytes;
    };
    return {{row(page0, rlo) + none, row(page1, min(rhi, 16)) + (rlo > 0 || rhi < 31)}};
  }
  // Rows [rlo, rhi] of a tile, the nearest of them for the others (PageTile::fetch).
  __device__ __forceinline__ void issue(uint32_t lds, const CacheRows<T>& cache, const Place& at, int rlo,
                                        int rhi) const {
    const char* const k = reinterpret_cast<const char*>(cache.k);
    const char* const v = reinterpret_cast<const char*>(cache.v);
    const bool whole = (at.half[1] & 1) == 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool second = first_row(i) >= 16;
      const long from = (second ? at.half[1] : at.half[0]) & ~1l;
      uint32_t offset = voff[i];
      if (!whole) {
        const int row = min(max(first_row(i) + lane / kChunks, rlo), rhi) - (second ? min(rhi, 16) : rlo);
        offset = (uint32_t)row * kRowBytes + chunk(i);
      }
      const uint32_t dst = lds + 1024u * (uint32_t)(i * (THREADS / 64) + wave);
      dma16s(k + from, offset, dst);
      dma16s(v + from, offset, dst + kTileBytes);
    }
  }
};

// A tile's keys as one wave's operands of the 16x16x32 score products, straight from their pages:
// lane (n, g) holds pieces of keys n and 16 + n. A piece is 16 bytes of cache: 8 elements, columns
// 32 c + 8 g on, one product's; or 16 of e4m3, columns 64 c + 16 g on, two products' (the
// contraction may take the columns in any order that the queries share).
template <typename T, typename C, int D> struct KeyPieces {
  static constexpr bool kQuantised = sizeof(C) == 1;
  static constexpr int kPieces = D / (kQuantised ? 64 : 32);
  u32x4 data[2][kPieces];
  uint32_t code[kQuantised ? 2 : 1];

  // Column of the queries that product ks takes, for lane group g.
  __device__ __forceinline__ static int column(int ks, int g) {
    return kQuantised ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g;
  }
  __device__ __forceinline__ void fetch(const CacheRows<C>& cache, int hk, int kv_heads, int page_shift, int k0,
                                        int rlo, int rhi, int page0, int page1, int n, int g) {
    const int page_rows = 1 << page_shift;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int row = min(max(16 * kb + n, rlo), rhi);  // (PageTile::fetch)
      const long head = (long)(row < 16 ? page0 : page1) * kv_heads + hk;
      const long line = (head << page_shift) + ((k0 + row) & (page_rows - 1));
      const C* src = cache.k + line * D + g * (kQuantised ? 16 : 8);
#pragma unroll
      for (int c = 0; c < kPieces; ++c)
        data[kb][c] = *reinterpret_cast<const u32x4*>(src + c * (kQuantised ? 64 : 32));
      if constexpr (kQuantised) code[kb] = cache.k_scale[line];
    }
  }
  __device__ __forceinline__ void fetch(const CacheRows<C>& cache, const HalfRows& rows, int n, int g) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const long line = rows.of(16 * kb + n);
      const C* src = cache.k + line * D + g * (kQuantised ? 16 : 8);
#pragma unroll
      for (int c = 0; c < kPieces; ++c)
        data[kb][c] = *reinterpret_cast<const u32x4*>(src + c * (kQuantised ? 64 : 32));
      if constexpr (kQuantised) code[kb] = cache.k_scale[line];
    }
  }
  __device__ __forceinline__ V8<T> operand(int kb, int ks) const {
    if constexpr (kQuantised) {
      const u32x4 x = data[kb][ks >> 1];
      const float scale = scale_of(code[kb]);
      const V4<T> a = dequantise4<T>(x[2 * (ks & 1)], scale), b = dequantise4<T>(x[2 * (ks & 1) + 1], scale);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return __builtin_bit_cast(V8<T>, data[kb][ks]);
    }
  }
};

// The keys that a tile of rows of one sequence reads, as 32-key tiles: those that are visible
// as sinks only, then those from its first row's window to its last row's position.
struct PageSpan {
  int sink_keys, sink_tiles;  // keys [0, sink_keys)
  int lo, hi;                 // keys [lo, hi)
  int start;                  // lo, down to a multiple of 16
  int tiles;

  __device__ __forceinline__ PageSpan(int first_pos, int last_pos, int length, int window, int sinks) {
    hi = max(0, min(length, last_pos + 1));
    lo = window ? min(max(0, first_pos - window + 1), hi) : 0;
    sink_keys = window ? max(0, min(sinks, lo)) : 0;
    sink_tiles = (sink_keys + 31) / 32;
    start = lo & ~15;
    tiles = sink_tiles + (hi - start + 31) / 32;
    if (hi == 0) tiles = sink_tiles = 0;
  }
  // First key of tile t, and the first and last of its rows that are read.
  __device__ __forceinline__ int key(int t) const { return t < sink_tiles ? 32 * t : start + 32 * (t - sink_tiles); }
  __device__ __forceinline__ int first_row(int t) const { return t < sink_tiles ? 0 : max(0, lo - key(t)); }
  __device__ __forceinline__ int last_row(int t) const {
    return min(31, (t < sink_tiles ? sink_keys : hi) - 1 - key(t));
  }
};

}  // namespace fhog
