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

// Workgroups of a launch along the tokens, each of which leaves parts of its own.
struct RotaryGrid {
  int tile;  // tokens at a time
  int groups;
};
// Tokens a tile: enough that their rows keep 256 threads busy, few enough that small calls fill the card.
inline RotaryGrid rotary_grid(long tokens, int compute_units) {
  const int tile = tokens >= 16l * 4 * compute_units ? 16 : tokens >= 4l * 4 * compute_units ? 4 : 1;
  const long tiles = (tokens + tile - 1) / tile, most = 8l * compute_units;
  return RotaryGrid{tile, (int)(tiles < most ? tiles : most)};
}

// The weights' gradients from the workgroups' parts of them (0 of them: zeros).
template <typename T>
hipError_t sum_rotary_weights(const float* parts, void* const out[2], const RotaryShape& s, int groups, hipStream_t stream);
template <typename T> hipError_t launch_rotary_fwd(const RotaryFwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t s);
template <typename T> hipError_t launch_rotary_bwd(const RotaryBwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t s);
template <typename T> hipError_t launch_rotary_bwdbwd(const RotaryBwdBwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t s);

}  // namespace fhog
