// Norms of queries and keys for each head, with the position rotation in the same pass, and their
// first and second derivatives (fhog_rotary.h).
//
// A row x of H values, r = (mean x^2 + eps)^-1/2, n = r x, y = R(n w), where R turns the pairs of the
// first columns by angles p f_i. With g = R^T dy and the row means C = <g w, n> / H:
//   dx = r (g w - C n),   dw = sum over rows g n;
// and with cotangents u of dx and z of dw, U = <u, n> / H, A = <u, g w> / H, Z = <z g, n> / H:
//   ddy = R(r w (u - U n) + z n)
//   dx2 = r^2 (n (3 C U - A) - U g w - C u) + r (z g - Z n)
//   dw2 = sum over rows r g (u - U n).
// Without norms r = 1 and n = x, and only the rotation remains.
//
// All of it is fp32 from the loaded values on, rounded once where a row is stored. Angles are formed
// in 64 bits, reduced to a part of a turn there, and only then taken to fp32: at position 10^5 fp32
// would leave 4 10^-3 of an angle. They belong to a token, not to a head: a workgroup forms those of
// its tokens once, in LDS.
//
// L neighbouring lanes hold a row, N pairs a lane: both partners of a rotation are in one lane, in
// two loads of N elements where the row allows them. Every row is read once and written
// once. The weights' gradients are summed in registers over a workgroup's rows, then over its threads,
// then by a small kernel over the workgroups, always in the same order.
#include "fhog_paged.h"
#include "fhog_rotary.h"

namespace fhog {

namespace {

constexpr int kThreads = 256;
constexpr int N = kRotaryPairs;
constexpr int kMostTile = 16;

// N pairs of a row, a lane's.
struct Pairs {
  float a[N], b[N];
};

// Where lane c of a row finds its pairs N c .. N c + N - 1. Columns behind the rotated ones are paired with
// their neighbours and turned by nothing.
// WIDE: head_dim and rotated are multiples of 2 N, and N elements of a row are aligned to their size. (us, forward / backward /
// double backward of 8002 tokens, 40 heads, wide and by elements because rows lie one element off: bf16 D128 32 / 53 / 97 and
// 49 / 77 / 151, D64 20 / 32 / 49 and 41 / 62 / 100, fp32 D128 63 / 110 / 143 and 109 / 146 / 240. By elements a lane's pieces
// are N loads and stores each, and instructions bound it, at 2 to 3.4 TB/s.)
template <bool WIDE> struct Columns {
  int head_dim, half, pair0;
  bool apart;  // partners are half the rotated columns apart
  __device__ __forceinline__ Columns(const RotaryShape& s, int c)
      : head_dim(s.head_dim), half(s.rotated / 2), pair0(N * c), apart(!s.interleaved && N * c < s.rotated / 2) {}
  __device__ __forceinline__ bool any() const { return 2 * pair0 < head_dim; }
  __device__ __forceinline__ int column(int i, int side, bool interleaved) const {
    const int p = pair0 + i;
    return p < half && !interleaved ? p + side * half : 2 * p + side;
  }
  // A lane's part of a row as it lies in memory, and as pairs.
  template <typename T> struct Raw {
    typedef T VN __attribute__((ext_vector_type(N)));
    VN lo, hi;
  };
  template <typename T> __device__ __forceinline__ Raw<T> fetch(const T* row, bool interleaved) const {
    Raw<T> x;
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < N; ++i) x.lo[i] = x.hi[i] = (T)0.f;
      if (any()) {
        x.lo = *reinterpret_cast<const typename Raw<T>::VN*>(row + (apart ? pair0 : 2 * pair0));
        x.hi = *reinterpret_cast<const typename Raw<T>::VN*>(row + (apart ? pair0 + half : 2 * pair0 + N));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ca = column(i, 0, interleaved), cb = column(i, 1, interleaved);
        x.lo[i] = ca < head_dim ? row[ca] : (T)0.f;
        x.hi[i] = cb < head_dim ? row[cb] : (T)0.f;
      }
    }
    return x;
  }
  template <typename T> __device__ __forceinline__ Pairs take(const Raw<T>& r) const {
    Pairs x;
    if (apart || !WIDE) {
#pragma unroll
      for (int i = 0; i < N; ++i) x.a[i] = (float)r.lo[i], x.b[i] = (float)r.hi[i];
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        x.a[i] = (float)r.lo[2 * i], x.b[i] = (float)r.lo[2 * i + 1];
        x.a[N / 2 + i] = (float)r.hi[2 * i], x.b[N / 2 + i] = (float)r.hi[2 * i + 1];
      }
    }
    return x;
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const Pairs& x, bool interleaved) const {
    if constexpr (WIDE) {
      if (!any()) return;
      typedef T VN __attribute__((ext_vector_type(N)));
      typedef float FN __attribute__((ext_vector_type(N)));
      FN lo, hi;
      if (apart) {
#pragma unroll
        for (int i = 0; i < N; ++i) lo[i] = x.a[i], hi[i] = x.b[i];
      } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          lo[2 * i] = x.a[i], lo[2 * i + 1] = x.b[i];
          hi[2 * i] = x.a[N / 2 + i], hi[2 * i + 1] = x.b[N / 2 + i];
        }
      }
      *reinterpret_cast<VN*>(row + (apart ? pair0 : 2 * pair0)) = __builtin_convertvector(lo, VN);
      *reinterpret_cast<VN*>(row + (apart ? pair0 + half : 2 * pair0 + N)) = __builtin_convertvector(hi, VN);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ca = column(i, 0, interleaved), cb = column(i, 1, interleaved);
        if (ca < head_dim) row[ca] = (T)x.a[i];
        if (cb < head_dim) row[cb] = (T)x.b[i];
      }
    }
  }
};

// A weight, or a cotangent of one: in T or, beside 2-byte rows, in fp32.
template <typename T, bool WIDE>
__device__ __forceinline__ Pairs load_weight(const Columns<WIDE>& at, const void* w, const RotaryShape& s, float none) {
  Pairs x;
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) x.a[i] = x.b[i] = none;
    return x;
  }
  const Columns<false> one(s, at.pair0 / N);  // (its own alignment is not known)
  return s.wide_weights ? one.take(one.fetch((const float*)w, s.interleaved)) : one.take(one.fetch((const T*)w, s.interleaved));
}

// Sum over the L lanes of a row, in all of them.
template <int L> __device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) x += __shfl_xor(x, d, 64);
  return x;
}

__device__ __forceinline__ float dot(const Pairs& x, const Pairs& y) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) sum = fmaf(x.a[i], y.a[i], fmaf(x.b[i], y.b[i], sum));
  return sum;
}

// cos and sin of a token's angles for a lane's pairs, and the rotations.
struct Turn {
  alignas(16) float c[N];
  alignas(16) float s[N];
  __device__ __forceinline__ Pairs there(const Pairs& x) const {
    Pairs y;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      y.a[i] = x.a[i] * c[i] - x.b[i] * s[i];
      y.b[i] = x.b[i] * c[i] + x.a[i] * s[i];
    }
    return y;
  }
  __device__ __forceinline__ Pairs back(const Pairs& y) const {
    Pairs x;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x.a[i] = y.a[i] * c[i] + y.b[i] * s[i];
      x.b[i] = y.b[i] * c[i] - y.a[i] * s[i];
    }
    return x;
  }
};

__device__ __forceinline__ double position(const RotaryShape& s, long token) {
  if (s.positions != nullptr) {
    const long at = s.position_rows > 1 ? token : token % s.tokens;
    return s.position_bytes == 8 ? (double)((const long*)s.positions)[at] : (double)((const int*)s.positions)[at];
  }
  if (s.lengths == nullptr) return (double)(token % s.tokens);
  const int t = (int)token;
  if (s.offsets == nullptr) return (double)s.lengths[t] - 1.0;
  const CacheShape c{nullptr, s.lengths, s.offsets, s.sequences, s.tokens, 0, 0, 0, 0};
  const int b = last_at_or_before(s.sequences, t, [&](int i) { return packed_begin(c, i); });
  const int begin = packed_begin(c, b), end = packed_begin(c, b + 1);
  return t < begin || t >= end ? 0.0 : (double)s.lengths[b] - (double)(end - t);
}

// The workgroup's tokens [first, first + count): their angles, kPairs a token, and where their rows begin.
template <int L> struct Tokens {
  static constexpr int kPairs = N * L;
  alignas(16) float c[kMostTile][kPairs];
  alignas(16) float s[kMostTile][kPairs];
  long from[kMostTile];
  __device__ __forceinline__ void form(const RotaryShape& shape, const RowStrides& stride, long first, int count) {
    if ((int)threadIdx.x < count) {
      const long token = first + threadIdx.x, b = shape.batch == 1 ? 0 : token / shape.tokens;
      from[threadIdx.x] = b * stride.batch + (token - b * shape.tokens) * stride.token;
    }
    for (int i = threadIdx.x; i < count * kPairs; i += kThreads) {
      const int token = i / kPairs, pair = i % kPairs;
      float cos = 1.f, sin = 0.f;
      if (2 * pair < shape.rotated) {
        const double turns = position(shape, first + token) * (double)shape.frequencies[pair] * 0.15915494309189535;
        sincospif((float)(2.0 * (turns - rint(turns))), &sin, &cos);
      }
      c[token][pair] = cos;
      s[token][pair] = sin;
    }
  }
  __device__ __forceinline__ Turn turn(int token, int lane) const {
    Turn t;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      *reinterpret_cast<f32x4*>(t.c + i) = *reinterpret_cast<const f32x4*>(&c[token][N * lane + i]);
      *reinterpret_cast<f32x4*>(t.s + i) = *reinterpret_cast<const f32x4*>(&s[token][N * lane + i]);
    }
    return t;
  }
};

// For every row that this thread's lane group has, of the workgroup's tiles: fetch(offset of the row in x, offset in
// contiguous tensors), a row ahead, and work(what it gave, offset in contiguous tensors, Turn).
template <int L, typename Fetch, typename Work>
__device__ __forceinline__ void for_rows(const RotaryShape& s, const RowStrides& stride, int which, int tile,
                                         Tokens<L>& held, Fetch&& fetch, Work&& work) {
  constexpr int kRows = kThreads / L;
  const int heads = s.heads[which], lane = threadIdx.x % L, group = threadIdx.x / L;
  const int step_t = kRows / heads, step_h = kRows - step_t * heads, t_first = group / heads, h_first = group - t_first * heads;
  const long tokens = (long)s.batch * s.tokens;
  for (long t0 = (long)blockIdx.x * tile; t0 < tokens; t0 += (long)gridDim.x * tile) {
    const int count = (int)(tokens - t0 < tile ? tokens - t0 : tile);
    __syncthreads();  // (the tile before is read)
    held.form(s, stride, t0, count);
    __syncthreads();
    int t = t_first, h = h_first;
    if (t >= count) continue;
    auto place = [&] { return ((t0 + t) * heads + h) * (long)s.head_dim; };
    auto ahead = fetch(held.from[t] + h * stride.head, place());
    // (every lane of a group takes the same way, so the sums' shuffles find each other)
    while (t < count) {
      const auto now = ahead;
      const int at = t;
      const long to = place();
      t += step_t, h += step_h;
      if (h >= heads) h -= heads, ++t;
      if (t < count) ahead = fetch(held.from[t] + h * stride.head, place());
      work(now, to, held.turn(at, lane));
    }
  }
}

// A workgroup's part of a weight's gradient: the sums of its threads that hold the same columns.
template <int L, bool WIDE>
__device__ __forceinline__ void leave_parts(const Columns<WIDE>& at, const RotaryShape& s, const Pairs& sum, float* part,
                                            float* box) {
  // Lanes with the same columns within a wave, then the waves, through LDS.
  Pairs x = sum;
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (int d = L; d < 64; d <<= 1) {
      x.a[i] += __shfl_xor(x.a[i], d, 64);
      x.b[i] += __shfl_xor(x.b[i], d, 64);
    }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __syncthreads();
  if (lane < L)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      box[(wave * L + lane) * 2 * N + i] = x.a[i];
      box[(wave * L + lane) * 2 * N + N + i] = x.b[i];
    }
  __syncthreads();
  if (threadIdx.x < L)
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      float y = 0.f;
      for (int w = 0; w < kThreads / 64; ++w) y += box[(w * L + threadIdx.x) * 2 * N + i];
      const int col = at.column(i % N, i / N, s.interleaved);
      if (col < s.head_dim) part[col] = y;
    }
}

template <typename T, int L, bool WIDE>
__global__ void __launch_bounds__(kThreads) rotary_fwd_kernel(RotaryFwdParams<T> p, int tile) {
  __shared__ Tokens<L> held;
  const int which = blockIdx.y;
  const Columns<WIDE> at(p.s, threadIdx.x % L);
  const Pairs w = load_weight<T>(at, p.weight[which], p.s, 1.f);
  const float inv = 1.f / (float)p.s.head_dim;
  const T* const rows = p.x[which];
  T* const out = p.y[which];
  auto fetch = [&](long from, long) { return at.fetch(rows + from, p.s.interleaved); };
  for_rows<L>(p.s, p.stride[which], which, tile, held, fetch, [&](const auto& raw, long to, const Turn& turn) {
    Pairs x = at.take(raw);
    if (p.s.norm) {
      const float r = rsqrtf(row_sum<L>(dot(x, x)) * inv + p.s.eps);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x.a[i] *= r * w.a[i];
        x.b[i] *= r * w.b[i];
      }
    }
    at.store(out + to, turn.there(x), p.s.interleaved);
  });
}

template <typename T, int L, bool WIDE>
__global__ void __launch_bounds__(kThreads) rotary_bwd_kernel(RotaryBwdParams<T> p, int tile) {
  __shared__ Tokens<L> held;
  __shared__ float box[kThreads / 64 * L * 2 * N];
  const int which = blockIdx.y;
  const Columns<WIDE> at(p.s, threadIdx.x % L);
  const Pairs w = load_weight<T>(at, p.weight[which], p.s, 1.f);
  const float inv = 1.f / (float)p.s.head_dim;
  const T* const rows = p.x[which];
  const T* const dy = p.dy[which];
  T* const dx = p.dx[which];
  Pairs sum{};
  struct Rows {
    typename Columns<WIDE>::template Raw<T> dy, x;
  };
  auto fetch = [&](long from, long to) {
    Rows r{at.fetch(dy + to, p.s.interleaved), {}};
    if (p.s.norm) r.x = at.fetch(rows + from, p.s.interleaved);
    return r;
  };
  for_rows<L>(p.s, p.stride[which], which, tile, held, fetch, [&](const Rows& raw, long to, const Turn& turn) {
    Pairs g = turn.back(at.take(raw.dy));
    if (p.s.norm) {
      Pairs n = at.take(raw.x);
      const float r = rsqrtf(row_sum<L>(dot(n, n)) * inv + p.s.eps);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        n.a[i] *= r;
        n.b[i] *= r;
        sum.a[i] = fmaf(g.a[i], n.a[i], sum.a[i]);
        sum.b[i] = fmaf(g.b[i], n.b[i], sum.b[i]);
        g.a[i] *= w.a[i];
        g.b[i] *= w.b[i];
      }
      const float C = row_sum<L>(dot(g, n)) * inv;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        g.a[i] = r * (g.a[i] - C * n.a[i]);
        g.b[i] = r * (g.b[i] - C * n.b[i]);
      }
    }
    at.store(dx + to, g, p.s.interleaved);
  });
  if (p.parts != nullptr && p.weight[which] != nullptr)
    leave_parts<L>(at, p.s, sum, p.parts + ((long)which * gridDim.x + blockIdx.x) * p.s.head_dim, box);
}

template <typename T, int L, bool WIDE>
__global__ void __launch_bounds__(kThreads) rotary_bwdbwd_kernel(RotaryBwdBwdParams<T> p, int tile) {
  __shared__ Tokens<L> held;
  __shared__ float box[kThreads / 64 * L * 2 * N];
  const int which = blockIdx.y;
  const Columns<WIDE> at(p.s, threadIdx.x % L);
  const Pairs w = load_weight<T>(at, p.weight[which], p.s, 1.f);
  const Pairs z = load_weight<T>(at, p.z[which], p.s, 0.f);
  const float inv = 1.f / (float)p.s.head_dim;
  const T* const rows = p.x[which];
  const T* const dy = p.dy[which];
  const T* const cot = p.u[which];
  Pairs sum{};
  struct Rows {
    typename Columns<WIDE>::template Raw<T> x, dy, u;
  };
  auto fetch = [&](long from, long to) {
    return Rows{at.fetch(rows + from, p.s.interleaved), at.fetch(dy + to, p.s.interleaved), at.fetch(cot + to, p.s.interleaved)};
  };
  for_rows<L>(p.s, p.stride[which], which, tile, held, fetch, [&](const Rows& raw, long to, const Turn& turn) {
    Pairs n = at.take(raw.x);
    const Pairs g = turn.back(at.take(raw.dy));
    const Pairs u = at.take(raw.u);
    const float r = rsqrtf(row_sum<L>(dot(n, n)) * inv + p.s.eps);
    Pairs gw, zg;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      n.a[i] *= r, n.b[i] *= r;
      gw.a[i] = g.a[i] * w.a[i], gw.b[i] = g.b[i] * w.b[i];
      zg.a[i] = g.a[i] * z.a[i], zg.b[i] = g.b[i] * z.b[i];
    }
    const float C = row_sum<L>(dot(gw, n)) * inv, U = row_sum<L>(dot(u, n)) * inv;
    const float A = row_sum<L>(dot(u, gw)) * inv, Z = row_sum<L>(dot(zg, n)) * inv;
    const float r2 = r * r, nn = r2 * (3.f * C * U - A) - r * Z;
    Pairs dd, d2;
    auto one = [&](float n1, float g1, float gw1, float zg1, float u1, float w1, float z1, float& dd1, float& d21,
                   float& sum1) {
      const float rest = u1 - U * n1;
      dd1 = r * w1 * rest + z1 * n1;
      d21 = nn * n1 - r2 * (U * gw1 + C * u1) + r * zg1;
      sum1 = fmaf(r * g1, rest, sum1);
    };
#pragma unroll
    for (int i = 0; i < N; ++i) {
      one(n.a[i], g.a[i], gw.a[i], zg.a[i], u.a[i], w.a[i], z.a[i], dd.a[i], d2.a[i], sum.a[i]);
      one(n.b[i], g.b[i], gw.b[i], zg.b[i], u.b[i], w.b[i], z.b[i], dd.b[i], d2.b[i], sum.b[i]);
    }
    at.store(p.ddy[which] + to, turn.there(dd), p.s.interleaved);
    at.store(p.dx2[which] + to, d2, p.s.interleaved);
  });
  if (p.parts != nullptr && p.weight[which] != nullptr)
    leave_parts<L>(at, p.s, sum, p.parts + ((long)which * gridDim.x + blockIdx.x) * p.s.head_dim, box);
}

// The workgroups' parts of both weights' gradients to one: a workgroup eight columns, whose
// threads take every 64th part and meet in LDS.
constexpr int kWeightThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kWeightThreads) rotary_weights_kernel(const float* parts, void* out_q, void* out_k, int groups,
                                                                        int head_dim, int wide_weights) {
  __shared__ float box[kWeightThreads];
  void* const out = blockIdx.y ? out_k : out_q;
  if (out == nullptr) return;
  constexpr int kWays = kWeightThreads / 8;
  const int col = 8 * (int)blockIdx.x + (int)threadIdx.x % 8, way = threadIdx.x / 8;
  const float* const from = parts + (long)blockIdx.y * groups * head_dim + min(col, head_dim - 1);
  float sum = 0.f;
#pragma unroll 8
  for (int i = way; i < groups; i += kWays) sum += from[(long)i * head_dim];
  box[threadIdx.x] = sum;
  for (int half = kWays / 2; half > 0; half /= 2) {
    __syncthreads();
    if (way < half) box[threadIdx.x] += box[threadIdx.x + 8 * half];
  }
  if (way > 0 || col >= head_dim) return;
  sum = box[threadIdx.x];
  if (wide_weights)
    ((float*)out)[col] = sum;
  else
    ((T*)out)[col] = (T)sum;
}

// f.template operator()<L, WIDE>() with the lanes that a row takes, N pairs each.
template <typename F> void with_lanes(int head_dim, bool wide, F&& f) {
  auto lanes = [&]<int L>() { wide ? f.template operator()<L, true>() : f.template operator()<L, false>(); };
  if (head_dim <= 64)
    lanes.template operator()<32 / N>();
  else if (head_dim <= 128)
    lanes.template operator()<64 / N>();
  else
    lanes.template operator()<128 / N>();
}

}  // namespace

template <typename T>
hipError_t sum_rotary_weights(const float* parts, void* const out[2], const RotaryShape& s, int groups, hipStream_t stream) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (out[0] == nullptr && out[1] == nullptr)) return e;
  hipLaunchKernelGGL((rotary_weights_kernel<T>), dim3((s.head_dim + 7) / 8, 2), dim3(kWeightThreads), 0, stream, parts, out[0],
                     out[1], groups, s.head_dim, s.wide_weights);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_rotary_fwd(const RotaryFwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t stream) {
  with_lanes(p.s.head_dim, wide, [&]<int L, bool WIDE>() {
    hipLaunchKernelGGL((rotary_fwd_kernel<T, L, WIDE>), dim3(g.groups, 2), dim3(kThreads), 0, stream, p, g.tile);
  });
  return hipGetLastError();
}

template <typename T>
hipError_t launch_rotary_bwd(const RotaryBwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t stream) {
  with_lanes(p.s.head_dim, wide, [&]<int L, bool WIDE>() {
    hipLaunchKernelGGL((rotary_bwd_kernel<T, L, WIDE>), dim3(g.groups, 2), dim3(kThreads), 0, stream, p, g.tile);
  });
  return sum_rotary_weights<T>(p.parts, p.dweight, p.s, g.groups, stream);
}

template <typename T>
hipError_t launch_rotary_bwdbwd(const RotaryBwdBwdParams<T>& p, const RotaryGrid& g, bool wide, hipStream_t stream) {
  with_lanes(p.s.head_dim, wide, [&]<int L, bool WIDE>() {
    hipLaunchKernelGGL((rotary_bwdbwd_kernel<T, L, WIDE>), dim3(g.groups, 2), dim3(kThreads), 0, stream, p, g.tile);
  });
  return sum_rotary_weights<T>(p.parts, p.dweight2, p.s, g.groups, stream);
}

#define FHOG_INST(T)                                                                                         \
  template hipError_t sum_rotary_weights<T>(const float*, void* const*, const RotaryShape&, int, hipStream_t); \
  template hipError_t launch_rotary_fwd<T>(const RotaryFwdParams<T>&, const RotaryGrid&, bool, hipStream_t);  \
  template hipError_t launch_rotary_bwd<T>(const RotaryBwdParams<T>&, const RotaryGrid&, bool, hipStream_t);  \
  template hipError_t launch_rotary_bwdbwd<T>(const RotaryBwdBwdParams<T>&, const RotaryGrid&, bool, hipStream_t);
FHOG_INST(__bf16)
FHOG_INST(_Float16)
FHOG_INST(float)
#undef FHOG_INST

}  // namespace fhog
