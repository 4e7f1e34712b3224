// plh_scan.hip -- the gated linear recurrence, forward, backward and for one token.
//
//   a_t = sigmoid(f_t)      c_t = a_t c_{t-1} + (1 - a_t) g_t      h_t = sigmoid(o_t) c_t   (or h_t = c_t)
//
// over gates [batch][time][parts H] in the order f, g, o (parts = 3, or 2 without output gate).  c is linear in
// c_{t-1}, so a run of steps is one affine map c -> A c + B, and maps compose: (A2, B2) after (A1, B1) is
// (A1 A2, A2 B1 + B2).  The gradient is the same recurrence backwards in time: with the gradient u_t = s_t dh_t that
// h_t hands to c_t and E_t the one that c_{t-1} gets,
//   D_t = u_t + E_{t+1}     E_t = a_t D_t     dg_t = (1 - a_t) D_t     df_t = a_t (1 - a_t) (c_{t-1} - g_t) D_t
//   do_t = s_t (1 - s_t) c_t dh_t             E_{T} = dc_n,  dc_0 = E_0
// A row of n < T steps is the recurrence with a_t = 1, g_t = 0 from step n on; h is 0 there.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "plh_ops.h"

namespace plh {
namespace {

// A workgroup of 256 threads carries a slab of 64 channels through time, 64 steps (a tile) at a time.  Channels are
// numbered row after row, n = b H + h, so that slabs are full whatever H is.  A thread has VEC neighbouring channels
// for 16 / VEC consecutive steps: 64 / VEC threads side by side read 64 channels of one step, the groups of so many
// threads are consecutive in time.
constexpr int kScanThreads = 256;
constexpr int kSlab = 64;
constexpr int kTile = 64;

// Workgroups that a launch should have at least: with fewer slabs than that the time axis is split into segments.
constexpr int kScanGroups = 512;

struct Split {
  int tiles;      // tiles of a row
  int seg_tiles;  // ... of a segment
  int segs;
};

int64_t slabs_of(int64_t batch, int64_t hidden) { return (batch * hidden + kSlab - 1) / kSlab; }

Split split_for(int64_t batch, int64_t seq_len, int64_t hidden) {
  Split s;
  s.tiles = (int)((seq_len + kTile - 1) / kTile);
  const int64_t slabs = std::max<int64_t>(slabs_of(batch, hidden), 1);
  const int want = (int)std::max<int64_t>(1, kScanGroups / slabs);
  s.seg_tiles = std::max(1, (s.tiles + want - 1) / want);
  s.segs = std::max(1, (s.tiles + s.seg_tiles - 1) / s.seg_tiles);
  return s;
}

template <typename T>
struct ScanArgs {
  const T* gates;
  int64_t stride_b, stride_t;  // elements
  int64_t channels;            // B H
  int T_, H, tiles, seg_tiles, segs;
  unsigned slabs;
  const int32_t* lengths;
  const float* c0;
  T* out;         // [B][T][H]
  float* c_n;     // [B][H]
  float* states;  // [tiles][B][H]: c before each tile, or null (backward: required)
  float *seg_a, *seg_b;  // [segs][B][H]: the segments' maps (segs > 1)
  const T* d_out;        // backward
  const float* d_cn;
  T* d_gates;  // [B][T][parts H]
  float* d_c0;
};

// Where a thread stands: its channels, its place among the time groups, its row's length.
template <int VEC>
struct Place {
  static constexpr int CT = kSlab / VEC;          // threads side by side
  static constexpr int TG = kScanThreads / CT;    // time groups
  static constexpr int R = kTile / TG;            // steps of a thread
  static constexpr int WG = kWave / CT;           // time groups of a wave
  int lane, wave, ct, tg;
  int64_t n;  // first channel
  bool on;
  int64_t b;
  int h, len;

  template <typename T>
  __device__ __forceinline__ Place(const ScanArgs<T>& p, unsigned slab) {
    const int tid = threadIdx.x;
    lane = tid % kWave, ct = tid % CT, tg = tid / CT;
    wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    n = (int64_t)slab * kSlab + ct * VEC;
    on = n < p.channels;
    b = 0, h = 0, len = 0;
    if (on) {
      b = (uint32_t)n / (uint32_t)p.H;  // (channels <= 2^29)
      h = (int)((uint32_t)n % (uint32_t)p.H);
      len = p.T_;
      if (p.lengths) len = min(max(p.lengths[b], 0), p.T_);
    }
  }
};

// v of the even and of the odd time group of a pair of groups, in both (one exchange per level and value).
template <int VEC, int LEVEL>
__device__ __forceinline__ void pair_of(float v, float& even, float& odd) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  uint32_t lo, hi;
  if constexpr (VEC == 4 && LEVEL == 0) {  // groups of 16 lanes: neighbouring rows
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    lo = r[0], hi = r[1];
  } else {  // halves of the wave
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    lo = r[0], hi = r[1];
  }
  even = __builtin_bit_cast(float, lo), odd = __builtin_bit_cast(float, hi);
}

// The maps of the time groups of a wave, composed.  In: a thread's own factor A and its own sums B[k] (k = 0: of its
// steps in order; k = 1: in reverse order, SUMS = 2 only).  Out: pa[k], pb[k], the map of everything in this wave
// that comes before the thread's steps in direction k (REVERSE0: direction 0 is reverse order too); A and B become the
// wave's own.
template <int VEC, int SUMS, bool REVERSE0>
__device__ __forceinline__ void wave_maps(int lane, float (&A)[VEC], float (&B)[SUMS][VEC], float (&pa)[SUMS][VEC],
                                          float (&pb)[SUMS][VEC]) {
  constexpr int kLevels = VEC == 4 ? 2 : VEC == 2 ? 1 : 0;
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) pa[k][j] = 1.0f, pb[k][j] = 0.0f;
  const auto level = [&](auto lv) {
    constexpr int L = decltype(lv)::value;
    const bool odd = (lane & (VEC == 4 && L == 0 ? 16 : 32)) != 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float a0, a1;
      pair_of<VEC, L>(A[j], a0, a1);
#pragma unroll
      for (int k = 0; k < SUMS; ++k) {
        const bool rev = REVERSE0 || k == 1;
        float b0, b1;
        pair_of<VEC, L>(B[k][j], b0, b1);
        // the other group of the pair comes first for the odd one in order, for the even one in reverse
        const float fa = rev ? a1 : a0, fb = rev ? b1 : b0, sa = rev ? a0 : a1, sb = rev ? b0 : b1;
        if (odd != rev) {
          pb[k][j] = fmaf(pa[k][j], fb, pb[k][j]);
          pa[k][j] *= fa;
        }
        B[k][j] = fmaf(sa, fb, sb);
      }
      A[j] = a0 * a1;
    }
  };
  if constexpr (kLevels >= 1) level(std::integral_constant<int, 0>());
  if constexpr (kLevels >= 2) level(std::integral_constant<int, 1>());
}

// The four waves' maps in LDS: [parity of the tile][wave][A, sums...][channel].  Two halves in turn need one barrier
// per tile: the half written next was last read before the barrier in between.
template <int SUMS>
using WaveMaps = float[2][kScanThreads / kWave][1 + SUMS][kSlab];

template <int VEC, int SUMS>
__device__ __forceinline__ void put_maps(const Place<VEC>& at, float (&lds)[kScanThreads / kWave][1 + SUMS][kSlab],
                                         const float (&A)[VEC], const float (&B)[SUMS][VEC]) {
  if (at.lane < Place<VEC>::CT) {
    Vec<float, VEC> v;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v.v[j] = A[j];
    store_vec(&lds[at.wave][0][at.ct * VEC], v);
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v.v[j] = B[k][j];
      store_vec(&lds[at.wave][1 + k][at.ct * VEC], v);
    }
  }
}

// The carry through the four waves' maps: `carry` becomes the value after the whole tile, `mine` the value that this
// thread's steps start from; (pa, pb) is the thread's map from wave_maps.
template <int VEC, int SUMS, int K, bool REVERSE>
__device__ __forceinline__ void fold_waves(const Place<VEC>& at, const float (&lds)[kScanThreads / kWave][1 + SUMS][kSlab],
                                           const float (&pa)[VEC], const float (&pb)[VEC], float (&carry)[VEC],
                                           float (&mine)[VEC]) {
  constexpr int W = kScanThreads / kWave;
  float before[VEC];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int w = REVERSE ? W - 1 - i : i;
    if (w == at.wave) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) before[j] = carry[j];
    }
    const Vec<float, VEC> a = load_vec<float, VEC>(&lds[w][0][at.ct * VEC]);
    const Vec<float, VEC> b = load_vec<float, VEC>(&lds[w][1 + K][at.ct * VEC]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) carry[j] = fmaf(a.v[j], carry[j], b.v[j]);
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) mine[j] = fmaf(pa[j], before[j], pb[j]);
}

// The carry at a segment's start: the maps of the segments before it, in order, applied to `carry`.
template <typename T, int VEC>
__device__ __forceinline__ void fold_segments(const ScanArgs<T>& p, const Place<VEC>& at, int from, int to, int step,
                                              float (&carry)[VEC]) {
  if (!at.on) return;
  for (int s = from; s != to; s += step) {
    const int64_t o = (int64_t)s * p.channels + at.n;
    const Vec<float, VEC> a = load_vec<float, VEC>(p.seg_a + o), b = load_vec<float, VEC>(p.seg_b + o);
#pragma unroll
    for (int j = 0; j < VEC; ++j) carry[j] = fmaf(a.v[j], carry[j], b.v[j]);
  }
}

// A thread's rows of a tile.  Steps past the row's length hold f = +inf, so that a = 1 and 1 - a = 0 without a test,
// and zeros.
template <typename T, int VEC, bool G, bool O, bool D>
struct Rows {
  static constexpr int R = Place<VEC>::R;
  Vec<T, VEC> f[R], g[R], o[R], d[R];

  __device__ __forceinline__ void load(const ScanArgs<T>& p, const Place<VEC>& at, int tile) {
    const int t0 = tile * kTile + at.tg * R;
    const T* src = p.gates + at.b * p.stride_b + (int64_t)t0 * p.stride_t + at.h;
    const T* grad = D ? p.d_out + (at.b * p.T_ + t0) * (int64_t)p.H + at.h : nullptr;
    const auto row = [&](int r) {
      f[r] = load_vec<T, VEC>(src);
      if (G) g[r] = load_vec<T, VEC>(src + p.H);
      if (O) o[r] = load_vec<T, VEC>(src + 2 * p.H);
      if (D) d[r] = load_vec<T, VEC>(grad);
    };
    if (__all(t0 + R <= at.len)) {  // (the usual case: no branch per row)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        row(r);
        src += p.stride_t;
        if (D) grad += p.H;
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          f[r].v[j] = (T)__builtin_inff();
          if (G) g[r].v[j] = (T)0.0f;
          if (O) o[r].v[j] = (T)0.0f;
          if (D) d[r].v[j] = (T)0.0f;
        }
        if (t0 + r < at.len) row(r);
        src += p.stride_t;
        if (D) grad += p.H;
      }
    }
  }
};

template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> zero_unless(bool live, const Vec<T, VEC>& v) {
  Vec<T, VEC> z;
#pragma unroll
  for (int j = 0; j < VEC; ++j) z.v[j] = live ? v.v[j] : (T)0.0f;
  return z;
}

template <int VEC>
__device__ __forceinline__ void load_carry(const float* src, const Place<VEC>& at, float (&c)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) c[j] = 0.0f;
  if (!src || !at.on) return;
  const Vec<float, VEC> v = load_vec<float, VEC>(src + at.n);
#pragma unroll
  for (int j = 0; j < VEC; ++j) c[j] = v.v[j];
}

template <int VEC>
__device__ __forceinline__ void store_carry(float* dst, const Place<VEC>& at, const float (&c)[VEC]) {
  Vec<float, VEC> v;
#pragma unroll
  for (int j = 0; j < VEC; ++j) v.v[j] = c[j];
  store_vec(dst + at.n, v);
}

// Forward.  MAPS: only the segments' maps (of all but the last), for the launch that follows.
template <typename T, int VEC, bool GATED, bool MAPS>
__global__ void __launch_bounds__(kScanThreads) scan_forward_kernel(ScanArgs<T> p) {
  using P = Place<VEC>;
  constexpr int R = P::R;
  __shared__ WaveMaps<1> lds;
  const unsigned slab = blockIdx.x % p.slabs;
  const int seg = blockIdx.x / p.slabs;
  const P at(p, slab);
  float carry[VEC], prod[VEC];
  load_carry<VEC>(MAPS ? nullptr : p.c0, at, carry);
  if (!MAPS) fold_segments<T, VEC>(p, at, 0, seg, 1, carry);
#pragma unroll
  for (int j = 0; j < VEC; ++j) prod[j] = 1.0f;
  const int tile_end = min(p.tiles, (seg + 1) * p.seg_tiles);
  Rows<T, VEC, true, GATED && !MAPS, false> x, next;
  int tile = seg * p.seg_tiles;
  if (tile < tile_end) next.load(p, at, tile);
  for (; tile < tile_end; ++tile) {
    x = next;
    if (tile + 1 < tile_end) next.load(p, at, tile + 1);
    const int t0 = tile * kTile + at.tg * R;
    float a[R][VEC], b[R][VEC], A[VEC], B[1][VEC], pa[1][VEC], pb[1][VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[0][j] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float ns;
        logistic((float)x.f[r].v[j], a[r][j], ns);
        b[r][j] = ns * (float)x.g[r].v[j];
        B[0][j] = fmaf(a[r][j], B[0][j], b[r][j]);
        A[j] *= a[r][j];
      }
    }
    wave_maps<VEC, 1, false>(at.lane, A, B, pa, pb);
    auto& maps = lds[tile & 1];
    put_maps<VEC, 1>(at, maps, A, B);
    __syncthreads();
    if (MAPS) {
#pragma unroll
      for (int w = 0; w < kScanThreads / kWave; ++w)
#pragma unroll
        for (int j = 0; j < VEC; ++j) prod[j] *= maps[w][0][at.ct * VEC + j];
    } else if (p.states && at.on && at.tg == 0) {
      store_carry<VEC>(p.states + (int64_t)tile * p.channels, at, carry);
    }
    float c[VEC];
    fold_waves<VEC, 1, 0, false>(at, maps, pa[0], pb[0], carry, c);
    if (!MAPS && at.on) {
      T* dst = p.out + (at.b * p.T_ + t0) * (int64_t)p.H + at.h;
      Vec<T, VEC> y[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          c[j] = fmaf(a[r][j], c[j], b[r][j]);
          y[r].v[j] = round_to<T>(GATED ? c[j] * sigmoid((float)x.o[r].v[j]) : c[j]);
        }
      }
      if (__all(t0 + R <= at.len)) {
#pragma unroll
        for (int r = 0; r < R; ++r) store_vec(dst + (int64_t)r * p.H, y[r]);
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (t0 + r < p.T_) store_vec(dst + (int64_t)r * p.H, zero_unless(t0 + r < at.len, y[r]));
      }
    }
  }
  if (at.on && at.tg == 0) {
    if (MAPS) {
      store_carry<VEC>(p.seg_a + (int64_t)seg * p.channels, at, prod);
      store_carry<VEC>(p.seg_b + (int64_t)seg * p.channels, at, carry);
    } else if (seg == p.segs - 1 && p.c_n) {
      store_carry<VEC>(p.c_n, at, carry);
    }
  }
}

// Backward: tiles from the last to the first.  MAPS: only the segments' maps of E (of all but the first).
template <typename T, int VEC, bool GATED, bool MAPS>
__global__ void __launch_bounds__(kScanThreads) scan_backward_kernel(ScanArgs<T> p) {
  using P = Place<VEC>;
  constexpr int R = P::R;
  constexpr int kParts = GATED ? 3 : 2;
  constexpr int kSums = MAPS ? 1 : 2;  // the sums in reverse order; else first those in order, for c
  constexpr int kRev = kSums - 1;
  __shared__ WaveMaps<kSums> lds;
  const unsigned slab = blockIdx.x % p.slabs;
  const int seg = blockIdx.x / p.slabs + (MAPS ? 1 : 0);
  const P at(p, slab);
  float carry[VEC], prod[VEC];
  load_carry<VEC>(MAPS ? nullptr : p.d_cn, at, carry);
  if (!MAPS) fold_segments<T, VEC>(p, at, p.segs - 1, seg, -1, carry);
#pragma unroll
  for (int j = 0; j < VEC; ++j) prod[j] = 1.0f;
  const int tile_first = seg * p.seg_tiles;
  Rows<T, VEC, !MAPS, GATED, true> x, next;
  float start[VEC], next_start[VEC];
  int tile = min(p.tiles, (seg + 1) * p.seg_tiles) - 1;
  if (tile >= tile_first) {
    next.load(p, at, tile);
    load_carry<VEC>(MAPS ? nullptr : p.states + (int64_t)tile * p.channels, at, next_start);
  }
  for (; tile >= tile_first; --tile) {
    x = next;
#pragma unroll
    for (int j = 0; j < VEC; ++j) start[j] = next_start[j];
    if (tile > tile_first) {
      next.load(p, at, tile - 1);
      load_carry<VEC>(MAPS ? nullptr : p.states + (int64_t)(tile - 1) * p.channels, at, next_start);
    }
    const int t0 = tile * kTile + at.tg * R;
    float a[R][VEC], na[R][VEC], u[R][VEC], w[R][VEC];  // a, 1 - a, u = s dh, w = (1 - s) u
    float A[VEC], B[kSums][VEC], pa[kSums][VEC], pb[kSums][VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[0][j] = B[kRev][j] = 0.0f;
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        logistic((float)x.f[r].v[j], a[r][j], na[r][j]);
        u[r][j] = (float)x.d[r].v[j];
        if (GATED) {
          float s, ns;
          logistic_fast((float)x.o[r].v[j], s, ns);
          u[r][j] *= s;
          w[r][j] = ns * u[r][j];
        }
        B[kRev][j] = a[r][j] * (B[kRev][j] + u[r][j]);
        A[j] *= a[r][j];
      }
    }
    if (!MAPS) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < VEC; ++j) B[0][j] = fmaf(a[r][j], B[0][j], na[r][j] * (float)x.g[r].v[j]);
    }
    wave_maps<VEC, kSums, MAPS>(at.lane, A, B, pa, pb);
    auto& maps = lds[tile & 1];
    put_maps<VEC, kSums>(at, maps, A, B);
    __syncthreads();
    if (MAPS) {
#pragma unroll
      for (int i = 0; i < kScanThreads / kWave; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) prod[j] *= maps[i][0][at.ct * VEC + j];
    }
    float e[VEC];
    fold_waves<VEC, kSums, kRev, true>(at, maps, pa[kRev], pb[kRev], carry, e);
    if (!MAPS && at.on) {
      // c before each of this thread's steps, from the state that the forward pass left at the tile's start
      float c[VEC], before[R][VEC];
      fold_waves<VEC, kSums, 0, false>(at, maps, pa[0], pb[0], start, c);
      Vec<T, VEC> df[R], dg[R], d_o[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          before[r][j] = c[j];
          c[j] = fmaf(a[r][j], c[j], na[r][j] * (float)x.g[r].v[j]);
          if (GATED) d_o[r].v[j] = round_to<T>(w[r][j] * c[j]);
        }
      }
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float D = u[r][j] + e[j];
          const float n = na[r][j] * D;
          e[j] = a[r][j] * D;
          dg[r].v[j] = round_to<T>(n);
          df[r].v[j] = round_to<T>(a[r][j] * n * (before[r][j] - (float)x.g[r].v[j]));
        }
      }
      T* const dst = p.d_gates + (at.b * p.T_ + t0) * (int64_t)(kParts * p.H) + at.h;
      const bool all = __all(t0 + R <= at.len);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        T* const q = dst + (int64_t)r * (kParts * p.H);
        if (all) {
          store_vec(q, df[r]);
          store_vec(q + p.H, dg[r]);
          if (GATED) store_vec(q + 2 * p.H, d_o[r]);
        } else if (t0 + r < p.T_) {
          const bool live = t0 + r < at.len;
          store_vec(q, zero_unless(live, df[r]));
          store_vec(q + p.H, zero_unless(live, dg[r]));
          if (GATED) store_vec(q + 2 * p.H, zero_unless(live, d_o[r]));
        }
      }
    }
  }
  if (at.on && at.tg == 0) {
    if (MAPS) {
      store_carry<VEC>(p.seg_a + (int64_t)seg * p.channels, at, prod);
      store_carry<VEC>(p.seg_b + (int64_t)seg * p.channels, at, carry);
    } else if (seg == 0 && p.d_c0) {
      store_carry<VEC>(p.d_c0, at, carry);
    }
  }
}

// One step of every row, for serving: a thread per VEC channels, nothing to scan.  (The tiled kernel would leave 63 of
// 64 steps idle: 20.4 us for 512 rows of 512 channels in bfloat16.)
template <typename T, int VEC, bool GATED>
__global__ void __launch_bounds__(kScanThreads) scan_step_kernel(ScanArgs<T> p) {
  const int64_t n = ((int64_t)blockIdx.x * kScanThreads + threadIdx.x) * VEC;
  if (n >= p.channels) return;
  const uint32_t b = (uint32_t)n / (uint32_t)p.H, h = (uint32_t)n % (uint32_t)p.H;  // (channels <= 2^29)
  Vec<float, VEC> c = {};
  if (p.c0) c = load_vec<float, VEC>(p.c0 + n);
  if (p.states) store_vec(p.states + n, c);
  Vec<T, VEC> y = {};
  if (!p.lengths || p.lengths[b] > 0) {
    const T* const src = p.gates + b * p.stride_b + h;
    const Vec<T, VEC> f = load_vec<T, VEC>(src), g = load_vec<T, VEC>(src + p.H);
    Vec<T, VEC> o = {};
    if (GATED) o = load_vec<T, VEC>(src + 2 * p.H);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float a, na;
      logistic((float)f.v[j], a, na);
      c.v[j] = fmaf(a, c.v[j], na * (float)g.v[j]);
      y.v[j] = round_to<T>(GATED ? c.v[j] * sigmoid((float)o.v[j]) : c.v[j]);
    }
  }
  if (p.c_n) store_vec(p.c_n + n, c);
  store_vec(p.out + n, y);
}

template <typename T, int VEC, bool GATED>
hipError_t launch_forward(const ScanArgs<T>& p, hipStream_t s) {
  if (p.T_ == 1) {
    const int64_t threads = (p.channels + VEC - 1) / VEC;
    hipLaunchKernelGGL((scan_step_kernel<T, VEC, GATED>), dim3((unsigned)((threads + kScanThreads - 1) / kScanThreads)),
                       dim3(kScanThreads), 0, s, p);
    return hipGetLastError();
  }
  if (p.segs > 1) {
    hipLaunchKernelGGL((scan_forward_kernel<T, VEC, GATED, true>), dim3(p.slabs * (unsigned)(p.segs - 1)),
                       dim3(kScanThreads), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((scan_forward_kernel<T, VEC, GATED, false>), dim3(p.slabs * (unsigned)p.segs), dim3(kScanThreads),
                     0, s, p);
  return hipGetLastError();
}

template <typename T, int VEC, bool GATED>
hipError_t launch_backward(const ScanArgs<T>& p, hipStream_t s) {
  if (p.segs > 1) {
    hipLaunchKernelGGL((scan_backward_kernel<T, VEC, GATED, true>), dim3(p.slabs * (unsigned)(p.segs - 1)),
                       dim3(kScanThreads), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((scan_backward_kernel<T, VEC, GATED, false>), dim3(p.slabs * (unsigned)p.segs), dim3(kScanThreads),
                     0, s, p);
  return hipGetLastError();
}

// Channels per thread: the widest of 4, 2 and 1 at which every access of a row is aligned.
template <typename T>
int scan_vec(const ScanArgs<T>& p) {
  for (int v : {4, 2})
    if (p.H % v == 0 && p.stride_b % v == 0 && p.stride_t % v == 0 && aligned<T>(p.gates, v) && aligned<T>(p.out, v) &&
        aligned<T>(p.d_out, v) && aligned<T>(p.d_gates, v) && aligned<float>(p.c0, v) && aligned<float>(p.c_n, v) &&
        aligned<float>(p.states, v) && aligned<float>(p.seg_a, v) && aligned<float>(p.seg_b, v) &&
        aligned<float>(p.d_cn, v) && aligned<float>(p.d_c0, v))
      return v;
  return 1;
}

template <typename T, bool BACKWARD>
hipError_t launch_scan(const ScanArgs<T>& p, bool gated, hipStream_t s) {
  const auto go = [&](auto vec) {
    constexpr int V = decltype(vec)::value;
    if constexpr (BACKWARD)
      return gated ? launch_backward<T, V, true>(p, s) : launch_backward<T, V, false>(p, s);
    else
      return gated ? launch_forward<T, V, true>(p, s) : launch_forward<T, V, false>(p, s);
  };
  switch (scan_vec(p)) {
    case 4: return go(std::integral_constant<int, 4>());
    case 2: return go(std::integral_constant<int, 2>());
    default: return go(std::integral_constant<int, 1>());
  }
}

// The checks that both directions share; PLH_OK or the error code.
int check_scan(const char* what, int dtype, const void* gates, int64_t stride_b, int64_t stride_t, int64_t batch,
               int64_t seq_len, int hidden, const void* workspace, int64_t workspace_bytes) noexcept {
  if (dtype != PLH_F16 && dtype != PLH_BF16 && dtype != PLH_F32)
    return op_error(PLH_ERR_INVALID, what, "dtype must be PLH_F16, PLH_BF16 or PLH_F32");
  if (batch < 0 || seq_len < 0) return op_error(PLH_ERR_INVALID, what, "batch and seq_len must be non-negative");
  if (hidden < 1 || hidden > (1 << 24)) return op_error(PLH_ERR_UNSUPPORTED, what, "hidden must lie in [1, 2^24]");
  if (seq_len > (1 << 30) || batch > (1 << 29) || batch * hidden > (1 << 29))
    return op_error(PLH_ERR_UNSUPPORTED, what, "seq_len must not exceed 2^30, batch * hidden not 2^29");
  if (batch > 0 && seq_len > 0 && !gates) return op_error(PLH_ERR_INVALID, what, "gates is required");
  if (stride_b < 0 || stride_t < 0) return op_error(PLH_ERR_INVALID, what, "strides must be non-negative");
  const int64_t need = plh_gated_scan_workspace_bytes(batch, seq_len, hidden);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return op_error(PLH_ERR_INVALID, what, "workspace missing or smaller than plh_gated_scan_workspace_bytes()");
  if (!aligned<float>(workspace, 4)) return op_error(PLH_ERR_INVALID, what, "workspace must be 16-byte aligned");
  return PLH_OK;
}

template <typename T>
ScanArgs<T> scan_args(const void* gates, int64_t stride_b, int64_t stride_t, int64_t batch, int64_t seq_len, int hidden,
                      const int32_t* lengths, void* workspace) {
  const Split sp = split_for(batch, seq_len, hidden);
  ScanArgs<T> p = {};
  p.gates = (const T*)gates;
  p.stride_b = stride_b, p.stride_t = stride_t;
  p.channels = batch * hidden;
  p.T_ = (int)seq_len, p.H = hidden;
  p.tiles = sp.tiles, p.seg_tiles = sp.seg_tiles, p.segs = sp.segs;
  p.slabs = (unsigned)slabs_of(batch, hidden);
  p.lengths = lengths;
  p.seg_a = (float*)workspace;
  p.seg_b = p.seg_a ? p.seg_a + (p.channels * sp.segs + 3) / 4 * 4 : nullptr;
  return p;
}

}  // namespace
}  // namespace plh

extern "C" {

int64_t plh_gated_scan_states(int64_t seq_len) { return seq_len < 0 ? -1 : (seq_len + plh::kTile - 1) / plh::kTile; }

int64_t plh_gated_scan_workspace_bytes(int64_t batch, int64_t seq_len, int hidden) {
  if (batch < 0 || seq_len < 0 || hidden < 1 || seq_len > (1 << 30) || batch > (1 << 29)) return -1;
  const plh::Split s = plh::split_for(batch, seq_len, hidden);
  if (s.segs <= 1) return 0;
  return 2 * ((batch * hidden * s.segs + 3) / 4 * 4) * (int64_t)sizeof(float);
}

int plh_gated_scan_forward(int dtype, int output_gate, const void* gates, int64_t stride_b, int64_t stride_t,
                           int64_t batch, int64_t seq_len, int hidden, const int32_t* lengths, const float* c0,
                           void* out, float* c_n, float* states, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  const char* const what = "gated_scan_forward";
  const int rc = plh::check_scan(what, dtype, gates, stride_b, stride_t, batch, seq_len, hidden, workspace,
                                 workspace_bytes);
  if (rc != PLH_OK) return rc;
  if (batch == 0) return PLH_OK;
  if (seq_len > 0 && !out) return plh::op_error(PLH_ERR_INVALID, what, "out is required");
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    auto p = plh::scan_args<T>(gates, stride_b, stride_t, batch, seq_len, hidden, lengths, workspace);
    p.c0 = c0, p.out = (T*)out, p.c_n = c_n, p.states = states;
    e = plh::launch_scan<T, false>(p, output_gate != 0, (hipStream_t)stream);
  });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

int plh_gated_scan_backward(int dtype, int output_gate, const void* gates, int64_t stride_b, int64_t stride_t,
                            int64_t batch, int64_t seq_len, int hidden, const int32_t* lengths, const float* states,
                            const void* d_out, const float* d_cn, void* d_gates, float* d_c0, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  const char* const what = "gated_scan_backward";
  const int rc = plh::check_scan(what, dtype, gates, stride_b, stride_t, batch, seq_len, hidden, workspace,
                                 workspace_bytes);
  if (rc != PLH_OK) return rc;
  if (batch == 0) return PLH_OK;
  if (seq_len > 0 && (!states || !d_out || !d_gates))
    return plh::op_error(PLH_ERR_INVALID, what, "states, d_out and d_gates are required");
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    auto p = plh::scan_args<T>(gates, stride_b, stride_t, batch, seq_len, hidden, lengths, workspace);
    p.states = const_cast<float*>(states), p.d_out = (const T*)d_out, p.d_cn = d_cn;
    p.d_gates = (T*)d_gates, p.d_c0 = d_c0;
    e = plh::launch_scan<T, true>(p, output_gate != 0, (hipStream_t)stream);
  });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

}  // extern "C"
