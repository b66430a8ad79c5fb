// Windowed attention where 32-row blocks have to spread over their workgroup: the forward, dQ and
// dK/dV with one block of 32 rows a workgroup, whose four waves take every fourth tile of the
// streamed side, each through a ring of its own (no barrier in the sweep), and add up their
// accumulators at the end, always in the same order.
//
// Two uses. Small grids: the kernels with 64 to 128 rows a workgroup leave most of the chip
// empty and walk a window's tiles one by one; here a block's chain is a quarter as long. And
// sinks: the queries that see one behind their window (SinkGrid) meet 32 keys or fewer, so
// that in a key-tiled workgroup all waves but one would idle.
//
// Sums and statistics are fp32; probabilities and score gradients enter the products over keys or
// queries in T, one rounding of half a step a term, as in the other kernels (the matrix instructions take both
// operands in it): for 2-byte types outputs are 1.2 to 1.5 times as far from 64 bits as with fp32 ones.
//
// 256-byte rows at most (2-byte types at D = 64 and 128, fp32 at 64). A wave's ring has two stages
// where they leave room for two workgroups on a CU, and where registers allow one anyway; else one
// stage and two workgroups, which hide each other's loads: causal N1000 window 256, H8 fp32 (256
// blocks) dK/dV 43.4 -> 36.9 us, H16 D128 bf16 (512) forward 26.6 -> 14.8, dQ 24.4 -> 19.8. (Eight
// waves a workgroup at fp32: 44.2; the blocks are bound by the CU's matrix rate, 256 operations a
// cycle.)
#include "fhog_device.h"
#include "fhog_params.h"

namespace fhog {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
template <typename T, int D> constexpr bool kNarrow = D * sizeof(T) <= 128;  // rows of 128 bytes

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A wave's ring of tiles of TENSORS tensors with the same rows, and of STATS rows of 32 fp32
// statistics behind them (256 bytes each). Tile i of the wave is in stage i % kStages.
template <typename T, int D, int TENSORS, int STATS, int STAGES>
struct WaveRing {
  typedef SwzTile<T, D> G;
  static constexpr int kTile = G::kElems * (int)sizeof(T);
  static constexpr int kStage = TENSORS * kTile + STATS * 256;
  static constexpr int kStages = STAGES;
  static constexpr int kBytes = kStages * kStage;
  static constexpr int kOps = TENSORS * G::kLoads + STATS;  // vector-memory operations of a tile
  uint32_t lds, row_bytes;
  int lane;
  TileDma<T, D> dma;

  __device__ __forceinline__ WaveRing(uint32_t lds_, uint32_t row_bytes_, int lane_)
      : lds(lds_), row_bytes(row_bytes_), lane(lane_) {
    dma.init(row_bytes, 32, lane);
  }
  __device__ __forceinline__ uint32_t stage(int i) const { return lds + (uint32_t)(i % kStages) * kStage; }
  // src[j]: first row of the tile in tensor j, of which nvalid exist (the last one stands in for
  // the others); stat[j]: the statistic of that row.
  __device__ __forceinline__ void issue(int i, const T* const (&src)[TENSORS], const float* const* stat, int nvalid) {
    const uint32_t dst = stage(i);
    if (nvalid >= 32) {
#pragma unroll
      for (int j = 0; j < TENSORS; ++j) dma.issue(dst + j * kTile, src[j]);
    } else {
      TileDma<T, D> part;
      part.init(row_bytes, nvalid, lane);
#pragma unroll
      for (int j = 0; j < TENSORS; ++j) part.issue(dst + j * kTile, src[j]);
    }
#pragma unroll
    for (int j = 0; j < STATS; ++j)
      dma4s(stat[j], 4u * (uint32_t)min(lane & 31, nvalid - 1), dst + TENSORS * kTile + 256 * j);
  }
  // Waits for the wave's tile i of `count`, of which i + 1 may be in flight.
  __device__ __forceinline__ void wait(int i, int count) const {
    if (kStages > 1 && i + 1 < count)
      wait_vmem_le<kOps>();
    else
      wait_vmem_le<0>();
    asm volatile("" ::: "memory");  // the tile's reads stay behind the wait
  }
  // Value r of a statistic in the accumulator layout: that of row 8 (r / 4) + 4 g + r % 4.
  __device__ __forceinline__ f32x4 stat(int i, int j, int a, int g) const {
    const uint32_t at = stage(i) + TENSORS * kTile + 256 * j + 4 * (8 * a + 4 * g);
    return *reinterpret_cast<const __attribute__((address_space(3))) f32x4*>((uintptr_t)at);
  }
};

// The waves' accumulators, DT * 4 pieces of four values a lane each, meet in LDS (all waves are
// behind a barrier, and the rings are free).
template <int DT> struct Box {
  float* at;
  __device__ __forceinline__ Box(char* lds, int lane) : at(reinterpret_cast<float*>(lds) + 4 * lane) {}
  __device__ __forceinline__ f32x4* piece(int wave, int i) const {
    return reinterpret_cast<f32x4*>(at + 256 * (wave * DT * 4 + i));
  }
  __device__ __forceinline__ void put(int wave, const f32x16 (&acc)[DT]) const {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *piece(wave, 4 * dt + a) = f32x4{acc[dt][4 * a], acc[dt][4 * a + 1], acc[dt][4 * a + 2], acc[dt][4 * a + 3]};
  }
  __device__ __forceinline__ f32x4 sum(int i) const {
    f32x4 x = *piece(0, i);
#pragma unroll
    for (int w = 1; w < kWaves; ++w) x += *piece(w, i);
    return x;
  }
  // Column of piece i for lane group g.
  __device__ __forceinline__ static int column(int i, int g) { return 32 * (i / 4) + 8 * (i % 4) + 4 * g; }
};

// ------------------------------------------------------------------ forward

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
few_fwd_kernel(FwdParams<T> p) {
  constexpr int KS = D / 16, DT = D / 32;
  typedef WaveRing<T, D, 2, 0, kNarrow<T, D> ? 2 : 1> Ring;
  constexpr int kLds = kWaves * (Ring::kBytes > DT * 4096 ? Ring::kBytes : DT * 4096);
  __shared__ __attribute__((aligned(1024))) char s_kv[kLds];
  __shared__ float s_ml[kWaves][32][2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, g = lane >> 5;
  const int nqb = (p.nq + 31) / 32;
  const int bh = blockIdx.x / nqb, q0 = 32 * (blockIdx.x % nqb);
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kv_heads);
  const long rs = (long)p.heads * D, rsk = (long)p.kv_heads * D;
  const long qbase = ((long)b * p.nq * p.heads + h) * D;
  const long kbase = ((long)b * p.nk * p.kv_heads + hk) * D;
  const int qi = q0 + n;
  const bool qvalid = qi < p.nq;
  const bool negate = p.scale < 0.f;  // fwd_kernel
  V8<T> qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = *reinterpret_cast<const V8<T>*>(p.q + qbase + (long)min(qi, p.nq - 1) * rs + 16 * ks + 8 * g);
    if (negate) qf[ks] = -qf[ks];
  }
  const KeyTiles<kWindow> tiles(p, q0, 32);
  const KeyBounds<kWindow> sees(p, q0, 32);
  const int count = tiles.count > wave ? (tiles.count - wave + kWaves - 1) / kWaves : 0;  // this wave's tiles
  SwzFrags<T, D> fr;
  fr.init(lane);
  Ring ring(lds_base_u32(s_kv) + wave * Ring::kBytes, (uint32_t)(rsk * (long)sizeof(T)), lane);
  auto issue = [&](int i) {
    const int kt = tiles.tile(wave + kWaves * i);
    const long off = kbase + (long)kt * 32 * rsk;
    const T* const src[2] = {p.k + off, p.v + off};
    ring.issue(i, src, nullptr, p.nk - 32 * kt);
  };
  const float c2 = fabsf(p.scale) * kLog2e;
  constexpr float kBound = 256.f;
  float m = -1e30f, lpart = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();
  wait_vmem();  // (fwd_kernel)
#pragma unroll
  for (int i = 0; i < Ring::kStages; ++i)
    if (i < count) issue(i);
  for (int i = 0; i < count; ++i) {
    ring.wait(i, count);
    const int kt = tiles.tile(wave + kWaves * i), k0 = 32 * kt;
    const uint32_t sa = ring.stage(i);
    f32x16 S = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) S = mma<T>(fr.rowf(sa, 0, ks), qf[ks], S);
    if (k0 + 32 > p.nk || k0 + 31 > q0 + p.coff || sees.below(k0)) {
      const int klim = min(p.nk - 1, qi + p.coff) - k0, klow = qi + p.coff - p.window + 1 - k0;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (crow(r, g) > klim || outside<kWindow>(crow(r, g), klow, p.sinks - k0)) S[r] = -INFINITY;
    }
    f32x16 P;
    auto probabilities = [&] {
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        P[r] = exp2_fast(fmaf(S[r], c2, -m));
        sum += P[r];
      }
      return sum;
    };
    float psum = probabilities();
    if (__any(!(psum <= kBound))) {  // the lazy rescale of fwd_kernel
      float top = S[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, S[r]);
      const float mnew = fmaxf(m, xgroup_max(top * c2));
      const float alpha = exp2_fast(m - mnew);
      lpart *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      m = mnew;
      psum = probabilities();
    }
    lpart += psum;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const V8<T> oP = cvt8<T>(s ? hi8(P) : lo8(P));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = mma<T>(fr.trf(sa, Ring::kTile, dt, s), oP, acc[dt]);
    }
    wait_lds();  // this stage's reads are done
    if (i + Ring::kStages < count) issue(i + Ring::kStages);
  }

  const float l = xgroup_sum(lpart);
  if (g == 0) {
    s_ml[wave][n][0] = m;
    s_ml[wave][n][1] = l;
  }
  __syncthreads();
  // Each wave's sums on the scale of the row's maximum; a row that sees nothing: O = 0, L = +inf.
  float top = s_ml[0][n][0], sum = 0.f;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_ml[w][n][0]);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += s_ml[w][n][1] * exp2_fast(s_ml[w][n][0] - top);
  const float f = sum > 0.f ? exp2_fast(m - top) / sum : 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
  const Box<DT> box(s_kv, lane);
  box.put(wave, acc);
  __syncthreads();
  if (!qvalid) return;
  for (int i = wave; i < DT * 4; i += kWaves)
    *reinterpret_cast<V4<T>*>(p.o + qbase + (long)qi * rs + Box<DT>::column(i, g)) = cvt4<T>(box.sum(i));
  if (wave == 0 && g == 0) p.lse[(long)bh * p.nq + qi] = sum > 0.f ? (top + __log2f(sum)) * kLn2 : INFINITY;
}

// ------------------------------------------------------------------ dQ and D

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
few_dq_kernel(BwdParams<T> p) {
  constexpr int KS = D / 16, DT = D / 32;
  typedef WaveRing<T, D, 2, 0, kNarrow<T, D> ? 2 : 1> Ring;
  constexpr int kLds = kWaves * (Ring::kBytes > DT * 4096 ? Ring::kBytes : DT * 4096);
  __shared__ __attribute__((aligned(1024))) char s_kv[kLds];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, g = lane >> 5;
  const int nqb = (p.nq + 31) / 32;
  const int bh = blockIdx.x / nqb, q0 = 32 * (blockIdx.x % nqb);
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kv_heads);
  const long rs = (long)p.heads * D, rsk = (long)p.kv_heads * D;
  const long qbase = ((long)b * p.nq * p.heads + h) * D;
  const long kbase = ((long)b * p.nk * p.kv_heads + hk) * D;
  const long sbase = (long)bh * p.nq;
  const int qi = q0 + n;
  const bool qvalid = qi < p.nq;
  V8<T> qf[KS], dof[KS];
  float dpart = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const long off = qbase + (long)min(qi, p.nq - 1) * rs + 16 * ks + 8 * g;
    qf[ks] = *reinterpret_cast<const V8<T>*>(p.q + off);
    dof[ks] = *reinterpret_cast<const V8<T>*>(p.dout + off);
    const V8<T> of = *reinterpret_cast<const V8<T>*>(p.o + off);
    if constexpr (sizeof(T) == 2) {
      dpart = dot8<T>(of, dof[ks], dpart);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dpart += (float)of[e] * (float)dof[ks][e];
    }
  }
  const float Di = xgroup_sum(dpart);
  const float nL2 = -p.lse[sbase + min(qi, p.nq - 1)] * kLog2e;
  const float c2 = p.scale * kLog2e;
  const KeyTiles<kWindow> tiles(p, q0, 32);
  const KeyBounds<kWindow> sees(p, q0, 32);
  const int count = tiles.count > wave ? (tiles.count - wave + kWaves - 1) / kWaves : 0;
  SwzFrags<T, D> fr;
  fr.init(lane);
  Ring ring(lds_base_u32(s_kv) + wave * Ring::kBytes, (uint32_t)(rsk * (long)sizeof(T)), lane);
  auto issue = [&](int i) {
    const int kt = tiles.tile(wave + kWaves * i);
    const long off = kbase + (long)kt * 32 * rsk;
    const T* const src[2] = {p.k + off, p.v + off};
    ring.issue(i, src, nullptr, p.nk - 32 * kt);
  };
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();
  wait_vmem();
#pragma unroll
  for (int i = 0; i < Ring::kStages; ++i)
    if (i < count) issue(i);
  for (int i = 0; i < count; ++i) {
    ring.wait(i, count);
    const int kt = tiles.tile(wave + kWaves * i), k0 = 32 * kt;
    const uint32_t sa = ring.stage(i);
    f32x16 S = zero16(), u;
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] = -Di;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      S = mma<T>(fr.rowf(sa, 0, ks), qf[ks], S);
      u = mma<T>(fr.rowf(sa, Ring::kTile, ks), dof[ks], u);
    }
    f32x16 P;
#pragma unroll
    for (int r = 0; r < 16; ++r) P[r] = exp2_fast(fmaf(S[r], c2, nL2));
    if (k0 + 32 > p.nk || k0 + 31 > q0 + p.coff || sees.below(k0)) {
      const int klim = min(p.nk - 1, qi + p.coff) - k0, klow = qi + p.coff - p.window + 1 - k0;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (crow(r, g) > klim || outside<kWindow>(crow(r, g), klow, p.sinks - k0)) P[r] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 vdS;
#pragma unroll
      for (int e = 0; e < 8; ++e) vdS[e] = P[8 * s + e] * u[8 * s + e];  // dS / scale
      const V8<T> oS = cvt8<T>(vdS);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = mma<T>(fr.trf(sa, 0, dt, s), oS, acc[dt]);
    }
    wait_lds();
    if (i + Ring::kStages < count) issue(i + Ring::kStages);
  }
  __syncthreads();
  const Box<DT> box(s_kv, lane);
  box.put(wave, acc);
  __syncthreads();
  if (!qvalid) return;
  for (int i = wave; i < DT * 4; i += kWaves)
    *reinterpret_cast<V4<T>*>(p.dq + qbase + (long)qi * rs + Box<DT>::column(i, g)) = cvt4<T>(box.sum(i) * p.scale);
  if (wave == 0 && g == 0) p.delta[sbase + qi] = Di;
}

// ------------------------------------------------------------------ dK and dV

// The 32-key block, (batch, key/value head) pair and part of a workgroup: part 0 of every block
// (none: ONLY_SINKS), then the sinks' chunks (SinkGrid).
struct FewBlock {
  int kb, bh, part = 0;
  template <typename P> __device__ __forceinline__ FewBlock(const P& p, bool only_sinks) {
    const int pairs = p.batch * p.kv_heads, blocks = (p.nk + 31) / 32;
    const int extra = (int)blockIdx.x - (only_sinks ? 0 : blocks * pairs);
    kb = blockIdx.x % blocks;
    bh = blockIdx.x / blocks;
    sink_workgroup(p.sink, extra, pairs, kb, bh, part);
  }
};

// Stores a block's two outputs, this wave's quarter of their pieces: box0 of `first` (dV), box1 of
// `second` (dK), times f; fp32 parts where the row is a sink's.
template <typename T, int D, typename P, int DT>
__device__ __forceinline__ void few_store(const P& p, const FewBlock& fb, const Box<DT>& box0, const Box<DT>& box1,
                                          T* first, T* second, float f0, float f1, int wave, int lane) {
  const int n = lane & 31, g = lane >> 5;
  const int kj = 32 * fb.kb + n;
  if (kj >= p.nk) return;
  const int sinks = min(p.sinks, p.nk), pairs = p.batch * p.kv_heads;
  const bool sink = kj < sinks && p.sink.chunks > 0;
  if (fb.part > 0 && !sink) return;
  const long row = (((long)(fb.bh / p.kv_heads) * p.nk + kj) * p.kv_heads + fb.bh % p.kv_heads) * D;
  float* parts = sink ? p.sink_parts + 2 * (((long)fb.part * pairs + fb.bh) * sinks + kj) * D : nullptr;
  for (int i = wave; i < DT * 4; i += kWaves) {
    const int col = Box<DT>::column(i, g);
    const f32x4 x = box0.sum(i) * f0, y = box1.sum(i) * f1;
    if (sink) {
      *reinterpret_cast<f32x4*>(parts + col) = x;
      *reinterpret_cast<f32x4*>(parts + D + col) = y;
    } else {
      *reinterpret_cast<V4<T>*>(first + row + col) = cvt4<T>(x);
      *reinterpret_cast<V4<T>*>(second + row + col) = cvt4<T>(y);
    }
  }
}

template <typename T, int D, bool ONLY_SINKS>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 ? 2 : 1)))
few_dkdv_kernel(BwdParams<T> p) {
  constexpr int KS = D / 16, DT = D / 32;
  typedef WaveRing<T, D, 2, 2, sizeof(T) == 2 ? 2 : 1> Ring;
  constexpr int kBox = kWaves * DT * 4096;
  constexpr int kLds = kWaves * Ring::kBytes > 2 * kBox ? kWaves * Ring::kBytes : 2 * kBox;
  __shared__ __attribute__((aligned(1024))) char s_q[kLds];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, g = lane >> 5;
  const FewBlock fb(p, ONLY_SINKS);
  const int b = fb.bh / p.kv_heads, hk = fb.bh % p.kv_heads;
  const int grp = p.heads / p.kv_heads;
  const long rs = (long)p.heads * D, rsk = (long)p.kv_heads * D;
  const long qbase = ((long)b * p.nq * p.heads + (long)hk * grp) * D;
  const long kbase = ((long)b * p.nk * p.kv_heads + hk) * D;
  const long sbase = ((long)b * p.heads + (long)hk * grp) * p.nq;
  const int k0 = 32 * fb.kb, kj = k0 + n;
  const QueryBounds<kWindow> qs(p, fb.kb, 32, fb.part, p.sink.step);
  const int qt_begin = qs.q_begin / 32, nqt = (qs.q_end + 31) / 32;
  const int total = __builtin_amdgcn_readfirstlane(nqt > qt_begin ? (nqt - qt_begin) * grp : 0);
  const int count = total > wave ? (total - wave + kWaves - 1) / kWaves : 0;

  V8<T> kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const long off = kbase + (long)min(kj, p.nk - 1) * rsk + 16 * ks + 8 * g;
    kf[ks] = *reinterpret_cast<const V8<T>*>(p.k + off);
    vf[ks] = *reinterpret_cast<const V8<T>*>(p.v + off);
  }
  const float c2 = p.scale * kLog2e;
  SwzFrags<T, D> fr;
  fr.init(lane);
  Ring ring(lds_base_u32(s_q) + wave * Ring::kBytes, (uint32_t)(rs * (long)sizeof(T)), lane);
  auto query_of = [&](int i) { return 32 * (qt_begin + (wave + kWaves * i) / grp); };
  auto issue = [&](int i) {
    const int q0 = query_of(i), gi = (wave + kWaves * i) % grp;
    const long off = qbase + (long)q0 * rs + (long)gi * D, soff = sbase + (long)gi * p.nq + q0;
    const T* const src[2] = {p.q + off, p.dout + off};
    const float* const stat[2] = {p.lse + soff, p.delta + soff};
    ring.issue(i, src, stat, p.nq - q0);
  };
  f32x16 acc_dk[DT], acc_dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc_dk[dt] = acc_dv[dt] = zero16();
  wait_vmem();
#pragma unroll
  for (int i = 0; i < Ring::kStages; ++i)
    if (i < count) issue(i);
  for (int i = 0; i < count; ++i) {
    ring.wait(i, count);
    const int q0 = query_of(i);
    const uint32_t sa = ring.stage(i);
    f32x16 S = zero16(), u;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 d = ring.stat(i, 1, a, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) u[4 * a + j] = -d[j];
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      S = mma<T>(fr.rowf(sa, 0, ks), kf[ks], S);
      u = mma<T>(fr.rowf(sa, Ring::kTile, ks), vf[ks], u);
    }
    f32x16 P;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 lse = ring.stat(i, 0, a, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) P[4 * a + j] = exp2_fast(fmaf(S[4 * a + j], c2, -lse[j] * kLog2e));
    }
    if (qs.masked(q0, k0)) {
      const int qlo = qs.lo(kj) - q0, qhi = qs.hi(kj) - q0;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = crow(r, g);
        if (m < qlo || m >= qhi) P[r] = 0.f;
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 vdS;
#pragma unroll
      for (int e = 0; e < 8; ++e) vdS[e] = P[8 * s + e] * u[8 * s + e];  // dS / scale
      const V8<T> oP = cvt8<T>(s ? hi8(P) : lo8(P)), oS = cvt8<T>(vdS);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        acc_dv[dt] = mma<T>(fr.trf(sa, Ring::kTile, dt, s), oP, acc_dv[dt]);
        acc_dk[dt] = mma<T>(fr.trf(sa, 0, dt, s), oS, acc_dk[dt]);
      }
    }
    wait_lds();
    if (i + Ring::kStages < count) issue(i + Ring::kStages);
  }
  __syncthreads();
  const Box<DT> box0(s_q, lane), box1(s_q + kBox, lane);
  box0.put(wave, acc_dv);
  box1.put(wave, acc_dk);
  __syncthreads();
  few_store<T, D>(p, fb, box0, box1, p.dv, p.dk, 1.f, p.scale, wave, lane);
}

// ------------------------------------------------------------------ dK2 and dV2

// Stage 2 of the double backward (fhog_bwdbwd_pair.hip).
template <typename T, int D, bool ONLY_SINKS>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1)))
few_stage2_kernel(BwdBwdParams<T> p) {
  constexpr int KS = D / 16, DT = D / 32;
  typedef WaveRing<T, D, 3, 4, kNarrow<T, D> ? 2 : 1> Ring;
  constexpr int kBox = kWaves * DT * 4096;
  constexpr int kLds = kWaves * Ring::kBytes > 2 * kBox ? kWaves * Ring::kBytes : 2 * kBox;
  __shared__ __attribute__((aligned(1024))) char s_q[kLds];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, g = lane >> 5;
  const FewBlock fb(p, ONLY_SINKS);
  const int b = fb.bh / p.kv_heads, hk = fb.bh % p.kv_heads;
  const int grp = p.heads / p.kv_heads;
  const long rs = (long)p.heads * D, rsk = (long)p.kv_heads * D;
  const long qbase = ((long)b * p.nq * p.heads + (long)hk * grp) * D;
  const long kbase = ((long)b * p.nk * p.kv_heads + hk) * D;
  const long sbase = ((long)b * p.heads + (long)hk * grp) * p.nq;
  const int k0 = 32 * fb.kb, kj = k0 + n;
  const QueryBounds<kWindow> qs(p, fb.kb, 32, fb.part, p.sink.step);
  const int qt_begin = qs.q_begin / 32, nqt = (qs.q_end + 31) / 32;
  const int total = __builtin_amdgcn_readfirstlane(nqt > qt_begin ? (nqt - qt_begin) * grp : 0);
  const int count = total > wave ? (total - wave + kWaves - 1) / kWaves : 0;

  V8<T> kf[KS], vf[KS], dkf[KS], dvf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const long off = kbase + (long)min(kj, p.nk - 1) * rsk + 16 * ks + 8 * g;
    kf[ks] = *reinterpret_cast<const V8<T>*>(p.k + off);
    vf[ks] = *reinterpret_cast<const V8<T>*>(p.v + off);
    dkf[ks] = *reinterpret_cast<const V8<T>*>(p.ddk + off);
    dvf[ks] = *reinterpret_cast<const V8<T>*>(p.ddv + off);
  }
  const float scale = p.scale, c2 = scale * kLog2e;
  SwzFrags<T, D> fr;
  fr.init(lane);
  Ring ring(lds_base_u32(s_q) + wave * Ring::kBytes, (uint32_t)(rs * (long)sizeof(T)), lane);
  auto query_of = [&](int i) { return 32 * (qt_begin + (wave + kWaves * i) / grp); };
  auto issue = [&](int i) {
    const int q0 = query_of(i), gi = (wave + kWaves * i) % grp;
    const long off = qbase + (long)q0 * rs + (long)gi * D, soff = sbase + (long)gi * p.nq + q0;
    const T* const src[3] = {p.q + off, p.dout + off, p.ddq + off};
    const float* const stat[4] = {p.lse + soff, p.delta + soff, p.ddelta + soff, p.bstat + soff};
    ring.issue(i, src, stat, p.nq - q0);
  };
  f32x16 acc_dk[DT], acc_dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc_dk[dt] = acc_dv[dt] = zero16();
  wait_vmem();
#pragma unroll
  for (int i = 0; i < Ring::kStages; ++i)
    if (i < count) issue(i);
  for (int i = 0; i < count; ++i) {
    ring.wait(i, count);
    const int q0 = query_of(i);
    const uint32_t sa = ring.stage(i);  // Q, dO, ddQ
    f32x16 S = zero16(), ddS = zero16(), u, dPa;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 d = ring.stat(i, 1, a, g), dd = ring.stat(i, 2, a, g), bst = ring.stat(i, 3, a, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u[4 * a + j] = -d[j];
        dPa[4 * a + j] = -fmaf(d[j], dd[j], bst[j]);
      }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const V8<T> qa = fr.rowf(sa, 0, ks), doa = fr.rowf(sa, Ring::kTile, ks), dqa = fr.rowf(sa, 2 * Ring::kTile, ks);
      S = mma<T>(qa, kf[ks], S);
      ddS = mma<T>(dqa, kf[ks], ddS);
      ddS = mma<T>(qa, dkf[ks], ddS);
      u = mma<T>(doa, vf[ks], u);        // dP - D
      dPa = mma<T>(doa, dvf[ks], dPa);   // dPa - (D dD + B)
    }
    f32x16 P, t;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 lse = ring.stat(i, 0, a, g), dd = ring.stat(i, 2, a, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * a + j;
        P[r] = exp2_fast(fmaf(S[r], c2, -lse[j] * kLog2e));
        t[r] = fmaf(ddS[r], scale, -dd[j]);  // ddS - dD
      }
    }
    // A query that sees one key adds nothing (first_contributing_query); none does at positions
    // from 1 to the last key if the window holds two.
    if (p.window == 1 || q0 + p.coff <= 0 || q0 + 31 + p.coff >= p.nk) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (keys_seen<kWindow>(p, q0 + crow(r, g)) == 1) P[r] = 0.f;
    }
    if (qs.masked(q0, k0)) {
      const int qlo = qs.lo(kj) - q0, qhi = qs.hi(kj) - q0;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = crow(r, g);
        if (m < qlo || m >= qhi) P[r] = 0.f;
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 vdS, vdS2, vddP;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = 8 * s + e;
        vdS[e] = P[r] * u[r];
        vdS2[e] = P[r] * fmaf(u[r], t[r], dPa[r]);  // P (dP2 - B)
        vddP[e] = P[r] * t[r];
      }
      const V8<T> oS = cvt8<T>(vdS), oS2 = cvt8<T>(vdS2), odP = cvt8<T>(vddP);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        acc_dk[dt] = mma<T>(fr.trf(sa, 2 * Ring::kTile, dt, s), oS, acc_dk[dt]);
        acc_dk[dt] = mma<T>(fr.trf(sa, 0, dt, s), oS2, acc_dk[dt]);
        acc_dv[dt] = mma<T>(fr.trf(sa, Ring::kTile, dt, s), odP, acc_dv[dt]);
      }
    }
    wait_lds();
    if (i + Ring::kStages < count) issue(i + Ring::kStages);
  }
  __syncthreads();
  const Box<DT> box0(s_q, lane), box1(s_q + kBox, lane);
  box0.put(wave, acc_dv);
  box1.put(wave, acc_dk);
  __syncthreads();
  few_store<T, D>(p, fb, box0, box1, p.dv2, p.dk2, 1.f, scale, wave, lane);
}

template <typename P> unsigned few_grid(const P& p, bool only_sinks) {
  return (unsigned)(key_grid<kWindow>(p, 32) - (only_sinks ? (p.nk + 31) / 32 * p.batch * p.kv_heads : 0));
}

}  // namespace

template <typename T, int D> hipError_t launch_few_fwd(const FwdParams<T>& p, hipStream_t stream) {
  hipLaunchKernelGGL((few_fwd_kernel<T, D>), dim3((p.nq + 31) / 32 * p.batch * p.heads), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}
template <typename T, int D> hipError_t launch_few_dq(const BwdParams<T>& p, hipStream_t stream) {
  hipLaunchKernelGGL((few_dq_kernel<T, D>), dim3((p.nq + 31) / 32 * p.batch * p.heads), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}
template <typename T, int D> hipError_t launch_few_dkdv(const BwdParams<T>& p, bool only_sinks, hipStream_t stream) {
  if (only_sinks)
    hipLaunchKernelGGL((few_dkdv_kernel<T, D, true>), dim3(few_grid(p, true)), dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((few_dkdv_kernel<T, D, false>), dim3(few_grid(p, false)), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}
template <typename T, int D> hipError_t launch_few_stage2(const BwdBwdParams<T>& p, bool only_sinks, hipStream_t stream) {
  if (only_sinks)
    hipLaunchKernelGGL((few_stage2_kernel<T, D, true>), dim3(few_grid(p, true)), dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((few_stage2_kernel<T, D, false>), dim3(few_grid(p, false)), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

#define FHOG_INST(T, D)                                                              \
  template hipError_t launch_few_fwd<T, D>(const FwdParams<T>&, hipStream_t);        \
  template hipError_t launch_few_dq<T, D>(const BwdParams<T>&, hipStream_t);         \
  template hipError_t launch_few_dkdv<T, D>(const BwdParams<T>&, bool, hipStream_t); \
  template hipError_t launch_few_stage2<T, D>(const BwdBwdParams<T>&, bool, hipStream_t);
FHOG_INST(__bf16, 64)
FHOG_INST(__bf16, 128)
FHOG_INST(_Float16, 64)
FHOG_INST(_Float16, 128)
FHOG_INST(float, 64)
#undef FHOG_INST

}  // namespace fhog
