// Which keys a query sees, as a template argument of the sequence-tiled kernels, and the
// tiles and bounds that a window of keys with sinks implies.
//
// MASK is 0 (every key), 1 (causal) or kWindow: a query at position p = i + coff sees the
// keys p - window < j <= p and, of the keys before those, the first `sinks`. In that mode a
// query block streams the tiles that hold its sinks and the tiles that its window touches,
// and a key block's queries are those from its diagonal to its window's end; a sink's
// queries behind its window are taken by workgroups of their own (SinkGrid).
#pragma once

#include <hip/hip_runtime.h>

namespace fhog {

constexpr int kWindow = 2;

// The 32-key tiles that a block of `rows` queries from q0 on streams: `sink_tiles` from the
// first one on, then those from `sink_tiles + jump` on. Iteration it takes tile(it).
template <int MASK> struct KeyTiles {
  int count;           // all of them
  int sink_tiles = 0;  // tiles before the window's first that hold sinks
  int jump = 0;

  template <typename P> __device__ __forceinline__ KeyTiles(const P& p, int q0, int rows) {
    int end = p.nk;
    if (MASK) end = min(end, q0 + rows + p.coff);
    const int nkt = end > 0 ? (end + 31) / 32 : 0;
    if constexpr (MASK == kWindow) {
      const int first = max(0, q0 + p.coff - p.window + 1) / 32;
      sink_tiles = min((min(p.sinks, p.nk) + 31) / 32, first);
      sink_tiles = __builtin_amdgcn_readfirstlane(nkt > 0 ? sink_tiles : 0);
      jump = __builtin_amdgcn_readfirstlane(first - sink_tiles);
      // (a block past all windows, top-left with nq > nk, has its sinks only)
      count = __builtin_amdgcn_readfirstlane(sink_tiles + max(0, nkt - first));
    } else {
      // (uniform; saying so keeps the compiler from treating the loop as divergent)
      count = __builtin_amdgcn_readfirstlane(nkt);
    }
  }
  __device__ __forceinline__ int tile(int it) const {
    if constexpr (MASK == kWindow) return it < sink_tiles ? it : it + jump;
    return it;
  }
};

// What 32 (or fewer) queries from q0 on see: tiles with work for them, tiles in which some
// pair is masked, and a query's bounds within a tile.
template <int MASK> struct KeyBounds {
  int end;        // tiles [0, end) hold a key at or before the last query's position
  int first = 0;  // first tile of the first query's window
  int wlow = 0;   // keys below this are outside the last query's window
  int sinks = 0;

  template <typename P> __device__ __forceinline__ KeyBounds(const P& p, int q0, int rows) {
    int wend = p.nk;
    if (MASK) wend = max(0, min(wend, q0 + rows + p.coff));
    end = q0 < p.nq ? (wend + 31) / 32 : 0;
    if constexpr (MASK == kWindow) {
      first = max(0, q0 + p.coff - p.window + 1) / 32;
      wlow = q0 + rows + p.coff - p.window;
      sinks = p.sinks;
    }
  }
  __device__ __forceinline__ bool active(int kt) const {
    if constexpr (MASK == kWindow) return kt < end && (kt >= first || 32 * kt < sinks);
    return kt < end;
  }
  // Whether a tile from k0 on (at or before the diagonal) holds keys outside some window.
  __device__ __forceinline__ bool below(int k0) const {
    return MASK == kWindow && k0 < wlow && k0 + 31 >= sinks;
  }
};

// The key at place m of a tile from k0 on is outside the window of the query whose window
// starts at key `low`, and no sink.
template <int MASK> __device__ __forceinline__ bool outside(int m, int low, int sinks) {
  return MASK == kWindow && m < low && m >= sinks;
}

// How many keys query qi sees.
template <int MASK, typename P> __device__ __forceinline__ int keys_seen(const P& p, int qi) {
  if constexpr (MASK == 0) return p.nk;
  const int hi = min(p.nk, qi + p.coff + 1);
  if constexpr (MASK != kWindow) return hi;
  const int low = max(0, qi + p.coff + 1 - p.window);  // its window starts here
  return max(0, hi - max(low, 0)) + max(0, min(p.sinks, min(low, hi)));
}

// The key-tiled kernels in window mode. Workgroups [0, blocks * pairs) take a block of
// `rows` keys each and the queries whose windows reach it; the others take a block that
// holds sinks and one chunk of the queries that see it as sinks only. A sink's row thus
// comes in parts, which go to p.sink_parts in fp32, part 0 from its own block and part
// 1 + c from chunk c, and sink_join adds them in that order.
struct SinkGrid {
  int blocks;  // key blocks that hold sinks (32-key ones: enough of any kernel's)
  int chunks;  // chunks of queries
  int step;    // queries of a chunk, a multiple of 32
  bool apart;  // whether the chunks have a launch of their own (sink_chunks)
};

// The block, (batch, head) pair and part of workgroup `extra` of those behind the ordinary ones
// (extra < 0: an ordinary one, which has them already).
__device__ __forceinline__ void sink_workgroup(const SinkGrid& sink, int extra, int pairs, int& kb, int& pair, int& part) {
  if (extra < 0) return;
  const int c = extra / pairs;
  pair = extra - c * pairs;
  part = 1 + c / sink.blocks;
  kb = c % sink.blocks;
}

// One workgroup's share of that grid: key block kb and queries [q_begin, q_end), of which
// key j takes [lo(j), hi(j)).
template <int MASK> struct QueryBounds {
  int q_begin, q_end, part = 0;
  int lo_add, hi_add, sink_end;  // lo = j + lo_add; hi = part ? nq if j < sink_end : j + hi_add
  int nq;

  template <typename P> __device__ __forceinline__ QueryBounds(const P& p, int kb, int rows, int chunk_part, int step) {
    nq = p.nq;
    if constexpr (MASK == kWindow) {
      part = chunk_part;
      sink_end = min(p.sinks, p.nk);
      lo_add = (part ? p.window : 0) - p.coff;
      hi_add = p.window - p.coff;
      const int first = max(0, kb * rows + lo_add) / 32 * 32;
      if (part == 0) {
        q_begin = first;
        q_end = max(0, min(nq, kb * rows + rows - 1 + hi_add));
      } else {
        // chunks count from the first query behind key 0's window
        q_begin = max(0, lo_add) / 32 * 32 + (part - 1) * step;
        q_end = min(nq, q_begin + step);
        q_begin = max(q_begin, first);
      }
    } else {
      q_begin = MASK ? max(0, kb * rows - p.coff) / 32 * 32 : 0;
      q_end = nq;
      lo_add = MASK ? -p.coff : 0;
      hi_add = sink_end = 0;
    }
  }
  __device__ __forceinline__ int lo(int j) const { return MASK ? j + lo_add : 0; }
  __device__ __forceinline__ int hi(int j) const {
    if constexpr (MASK != kWindow) return nq;
    return part ? (j < sink_end ? nq : 0) : min(nq, j + hi_add);
  }
  // Whether 32 queries from q0 on have work for 32 keys from k0 on, and whether some pair of
  // them is masked.
  __device__ __forceinline__ bool active(int q0, int k0) const {
    if constexpr (MASK == kWindow) return q0 + 31 >= lo(k0) && q0 < (part ? hi(k0) : hi(k0 + 31));
    return !MASK || q0 + 31 >= lo(k0);
  }
  __device__ __forceinline__ bool masked(int q0, int k0) const {
    if constexpr (MASK == kWindow)
      return q0 < lo(k0 + 31) || q0 + 32 > (part ? hi(k0 + 31) : hi(k0));
    return q0 + 32 > nq || (MASK && q0 < lo(k0 + 31));
  }
};

}  // namespace fhog
