// Norms of queries and keys for each head with the position rotation, and their first and
// second derivatives: parameter blocks (fhog_rotary.hip).
#pragma once

#include "fhog_device.h"

namespace fhog {

// Where a tensor's rows lie, in elements: a row of head_dim is contiguous.
struct RowStrides {
  long batch, token, head;
};

struct RotaryShape {
  int batch, tokens, heads[2], head_dim;  // heads: of queries and keys
  int rotated;                            // columns that turn: the first `rotated`
  int interleaved;                        // pairs (2 i, 2 i + 1), else (i, i + rotated / 2)
  int norm, wide_weights;                 // wide_weights: fp32 ones beside 2-byte rows
  float eps;
  const float* frequencies;  // (rotated / 2) radians a position
  // Positions: a tensor (batch, tokens) or (tokens), or a cache's lengths (sequences; the tokens are
  // packed as CacheShape says, batch 1), or neither: 0 on.
  const void* positions;
  int position_bytes, position_rows;
  const int* lengths;
  const int* offsets;
  int sequences;
};

// Each array: of queries, of keys.
template <typename T> struct RotaryFwdParams {
  const T* x[2];
  const void* weight[2];  // null: ones
  T* y[2];
  RowStrides stride[2];  // of x
  RotaryShape s;
};

template <typename T> struct RotaryBwdParams {
  const T* x[2];
  const void* weight[2];
  const T* dy[2];  // contiguous, as everything but x
  T* dx[2];
  float* parts;  // fp32 parts of the weights' gradients (2, workgroups, head_dim)
  void* dweight[2];
  RowStrides stride[2];
  RotaryShape s;
};

template <typename T> struct RotaryBwdBwdParams {
  const T* x[2];
  const void* weight[2];
  const T* dy[2];
  const T* u[2];     // cotangents of dx
  const void* z[2];  // of dweight (null where there is no weight)
  T* dx2[2];
  T* ddy[2];
  float* parts;
  void* dweight2[2];
  RowStrides stride[2];
  RotaryShape s;
};

// Pairs a lane. (Eight / four, us: forward of 8002 tokens, 40 heads of 128 fp16 35.0 / 34.6, its backward 57.7 / 55.7, the
// double backward of 16384 tokens, 24 heads of 64 bf16 82.6 / 66.6, with 195 and 119 registers.)
constexpr int kRotaryPairs = 4;

// Workgroups of a launch along the tokens (for queries, and as many for keys), each of which leaves parts of
// its own.
struct RotaryGrid {
  int tile;  // tokens at a time
  int groups;
};
// Tokens a tile: as many as leave four workgroups a CU, up to 16; but enough that their rows keep the threads busy.
inline RotaryGrid rotary_grid(long tokens, int heads, int head_dim, int compute_units) {
  const int cus = compute_units > 0 ? compute_units : 256, lanes = (head_dim <= 64 ? 32 : head_dim <= 128 ? 64 : 128) / kRotaryPairs;
  int tile = 1;
  while (tile < 16 && (tokens >= 4l * tile * cus || (tile < tokens && tile * heads * lanes < 256))) tile *= 2;
  const long tiles = (tokens + tile - 1) / tile, most = 4l * cus;
  return RotaryGrid{tile, (int)(tiles < most ? tiles : most)};
}

// The weights' gradients from the workgroups' parts of them (0 of them: zeros).
template <typename T>
hipError_t sum_rotary_weights(const float* parts, void* const out[2], const RotaryShape& s, int groups, hipStream_t stream);
template <typename T> hipError_t launch_rotary_fwd(const RotaryFwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t s);
template <typename T> hipError_t launch_rotary_bwd(const RotaryBwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t s);
template <typename T> hipError_t launch_rotary_bwdbwd(const RotaryBwdBwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t s);

}  // namespace fhog
