// plh_selective.hip -- the selective state space scan, forward, backward and for one token.
//
//   dt = softplus(raw + bias)    a_n = exp(dt A_n)    h_n <- a_n h_n + dt u B_n    y = sum_n C_n h_n + D u
//   out = y silu(z)
//
// per row b and channel d, n = 1 .. N states: u, raw and z are [batch][time][channels], B and C [batch][time][N] (the same
// for all channels), A [channels][N].  h is linear in what it was, so that a run of steps is one affine map per state,
// (P, Q): h -> P h + Q with P = exp(A sum dt), and maps compose.  Gradients, with dy = dout silu(z) and G_t the one that
// reaches h_t:
//   G_t = dy_t C_t + E_{t+1}      E_t = a_t G_t      (E_T = dh_n, dh_0 = E_0: the same recurrence backwards in time)
//   dC_t = sum_d dy_t h_t      dB_t = sum_d G_t dt u      s1 = sum_n G B      m = E_t h_{t-1}      s2 = sum_n m A
//   du = dt s1 + dy D      draw = (u s1 + s2) sigmoid(raw + bias)      dA = sum_{b,t} m dt      dD = sum_{b,t} dy u
//   dz = dout y silu'(z)      dbias = sum_{b,t} draw
// A row of len < T steps is the recurrence with dt = 0 (a = 1) and B = C = 0 from step len on.
//
// What bounds it: per state and step one exponential and four other operations forward (eight more backward, and
// the sums over states and channels), per channel and step four values of the activations' type forward, seven
// backward.  With 16 states the arithmetic takes longer than the traffic, so the layout saves operations: a thread has
// two neighbouring channels by four neighbouring states, whose B and C it reads once for both, and eight consecutive steps,
// whose decays stay in registers between the passes over them:
//   1. the decays, and the map of the thread's eight steps
//   2. the waves of a workgroup are consecutive in time; their maps meet in LDS around one barrier, and every wave folds
//      those before it into its own start
//   3. the eight steps from there, with the outputs
// so that an exponential is taken once although four times as many waves run as there are channels for.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "plh_ops.h"

namespace plh {
namespace {

constexpr int kCh = 2, kNs = 4;      // channels and states of a thread
constexpr int kSlots = kCh * kNs;
constexpr int kRun = 8;              // steps of a thread
constexpr int kWaves = 4;            // waves along time
constexpr int kTileSteps = kRun * kWaves;
constexpr int kMaxStates = 64;

struct Strided {  // [batch][time][...], dense in the last dimension; strides in elements
  const void* p;
  int64_t b, t;
};

struct SelArgs {
  Strided u, dt, z, B, C;  // z.p may be null
  const void *A, *D, *bias;  // [D][N], [D], [D]; D and bias may be null
  bool w32, softplus;
  const int32_t* lengths;
  const float* h0;  // [B][D][N] or null
  int64_t batch;
  int T_, D_, N;
  int groups;             // of channels, in a row
  int64_t units;          // groups of all rows
  int tiles, seg_tiles, segs;
  void* out;              // [B][T][D]
  float* h_n;             // [B][D][N] or null
  float* states;          // [tiles][B][D][N]: h before each tile, or null (backward: required)
  float* seg;             // [segs][2][B][D][N]: the segments' maps (segs > 1)
  const void* d_out;      // backward
  const float* d_hn;
  void *d_u, *d_dt, *d_z;  // [B][T][D]
  float* d_h0;
  float* part_bc;         // [bc_groups][B][T][2 N]: sums of dB and dC over the channels of a workgroup
  int bc_groups;
  float* part_w;          // [segs][B][D N + 2 D]: dA, dD, dbias
};

// Lanes of a wave: SL threads side by side have the states of a pair of channels, 64 / SL such pairs make a group.
template <int SL>
struct Wave {
  static constexpr int PAIRS = 64 / SL, CH = PAIRS * kCh, NP = SL * kNs;  // channels, padded states
  // How the wave reads its eight steps of CH channels: eight lanes per step with E neighbouring channels each.
  static constexpr int E = CH / 8;
  static_assert(kRun == 8 && CH % 8 == 0, "eight steps by eight lanes");
};

// Orders the LDS accesses of a wave's lanes among each other (they run in order; this is for the compiler).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

struct alignas(16) F4 {
  float v[4];
};
struct alignas(8) F2 {
  float v[2];
};

// Up to E elements, the first n of them from memory; the others zero.
template <typename T, int E>
__device__ __forceinline__ Vec<T, E> load_some(const T* p, int n) {
  Vec<T, E> v = {};
  if (n >= E) {
    v = load_vec<T, E>(p);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n) v.v[j] = p[j];
  }
  return v;
}
template <typename T, int E>
__device__ __forceinline__ void store_some(T* p, const Vec<T, E>& v, int n) {
  if (n >= E) {
    store_vec(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n) p[j] = v.v[j];
  }
}

template <typename T>
__device__ __forceinline__ float param(const void* p, bool p32, int64_t i, float fill) {
  return !p ? fill : p32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}

// log(1 + exp(v)) = max(v, 0) + log1p(exp(-|v|)) with log1p(e) = 2 artanh(s), s = e / (2 + e) in [0, 1/3]: the
// logarithm of a number close to one would lose the small values, which step sizes are.  The series' remainder after
// s^15 / 15 is below 2 s^17 / 17 / (1 - s^2) < 2^-29 s.
__device__ __forceinline__ float softplus_of(float v) {
  const float e = __builtin_amdgcn_exp2f(-__builtin_fabsf(v) * kOpLog2e);
  const float d = 2.0f + e, r = __builtin_amdgcn_rcpf(d), s = e * fmaf(fmaf(-d, r, 1.0f), r, r), q = s * s;
  float t = 1.0f / 15;
  t = fmaf(t, q, 1.0f / 13);
  t = fmaf(t, q, 1.0f / 11);
  t = fmaf(t, q, 1.0f / 9);
  t = fmaf(t, q, 1.0f / 7);
  t = fmaf(t, q, 1.0f / 5);
  t = fmaf(t, q, 1.0f / 3);
  t = fmaf(t * q, s, s);
  return fmaf(2.0f, t, __builtin_elementwise_maximum(v, 0.0f));
}

// The decay of a run of steps.  Every step's own is positive; their product may underflow (or, of a growing state,
// overflow), and 0 * inf would be NaN where the steps one after the other are not.
__device__ __forceinline__ float run_decay(float log2_decay) {
  return __builtin_amdgcn_exp2f(fminf(fmaxf(log2_decay, -126.0f), 127.0f));
}

// Sum over the SL lanes that share a pair of channels, to all of them.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  const int u = __builtin_bit_cast(int, v);
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, CTRL, 0xf, 0xf, true));
}
template <int SL>
__device__ __forceinline__ float states_sum(float v) {
  if constexpr (SL >= 2) v = add_dpp<0xB1>(v);   // quad_perm 1 0 3 2
  if constexpr (SL >= 4) v = add_dpp<0x4E>(v);   // quad_perm 2 3 0 1
  if constexpr (SL >= 8) v = add_dpp<0x141>(v);  // row_half_mirror
  if constexpr (SL >= 16) v = add_dpp<0x128>(v);  // row_ror 8
  return v;
}

// Sum of two values over the two halves of the wave, or of neighbouring rows of 16 lanes: the first value's in the low
// half (even row), the second's in the other.
template <bool HALVES>
__device__ __forceinline__ float pair_sum(float v0, float v1) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v0), b = __builtin_bit_cast(uint32_t, v1);
  if constexpr (HALVES) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
}
// Within a row of 16 lanes: over the lanes that differ in the bits above SL's.
template <int SL>
__device__ __forceinline__ float row_rest_sum(float v) {
  if constexpr (SL <= 8) v = add_dpp<0x128>(v);  // row_ror 8, 4, 2, 1
  if constexpr (SL <= 4) v = add_dpp<0x124>(v);
  if constexpr (SL <= 2) v = add_dpp<0x122>(v);
  if constexpr (SL <= 1) v = add_dpp<0x121>(v);
  return v;
}

// Where a wave stands: row, first channel of its group, its place in time.
struct At {
  int64_t b;
  int c0, len;
  bool on;
};
__device__ __forceinline__ At place(const SelArgs& p, int64_t unit, int channels) {
  At a;
  a.on = unit < p.units;
  a.b = a.on ? unit / p.groups : 0;
  a.c0 = a.on ? (int)(unit % p.groups) * channels : p.D_;
  a.len = 0;
  if (a.on) a.len = p.lengths ? min(max(p.lengths[a.b], 0), p.T_) : p.T_;
  return a;
}

// The LDS of a wave.
template <int SL>
struct WaveLds {
  F4 step[kRun][Wave<SL>::PAIRS];   // dt, dt u of the pair's two channels
  F4 bc[kRun][2][SL];               // B and C
  float y[kRun][Wave<SL>::CH];
};
struct MapLds {
  F4 v[kSlots / 4][64];
};

// A wave's states of the pair's two channels, [B][D][N] at row b; zero outside.
template <int SL>
struct Slots {
  int c, n;      // first channel and state
  int channels;  // of the two that there are
  __device__ __forceinline__ Slots(const SelArgs& p, const At& at, int lane) {
    c = at.c0 + lane / SL * kCh, n = lane % SL * kNs;
    channels = min(max(p.D_ - c, 0), kCh);
  }
  __device__ __forceinline__ void load(const SelArgs& p, const float* base, int64_t b, float (&v)[kSlots]) const {
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
      Vec<float, kNs> t = {};
      if (i < channels && n < p.N) t = load_some<float, kNs>(base + (b * p.D_ + c + i) * p.N + n, p.N - n);
#pragma unroll
      for (int j = 0; j < kNs; ++j) v[i * kNs + j] = t.v[j];
    }
  }
  __device__ __forceinline__ void store(const SelArgs& p, float* base, int64_t b, const float (&v)[kSlots]) const {
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
      Vec<float, kNs> t;
#pragma unroll
      for (int j = 0; j < kNs; ++j) t.v[j] = v[i * kNs + j];
      if (i < channels && n < p.N) store_some<float, kNs>(base + (b * p.D_ + c + i) * p.N + n, t, p.N - n);
    }
  }
};

__device__ __forceinline__ void put_map(MapLds& m, int lane, const float (&v)[kSlots]) {
#pragma unroll
  for (int q = 0; q < kSlots / 4; ++q) m.v[q][lane] = F4{{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]}};
}
__device__ __forceinline__ void get_map(const MapLds& m, int lane, float (&v)[kSlots]) {
#pragma unroll
  for (int q = 0; q < kSlots / 4; ++q) {
    const F4 t = m.v[q][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * q + j] = t.v[j];
  }
}

// A wave's eight steps of one activation tensor, as loaded.
template <typename T, int SL>
struct Rows {
  static constexpr int E = Wave<SL>::E;
  Vec<T, E> v;
  __device__ __forceinline__ void load(const Strided& s, const At& at, int t, int c, int n) {
    v = Vec<T, E>{};
    if (t < at.len && n > 0) v = load_some<T, E>(static_cast<const T*>(s.p) + at.b * s.b + (int64_t)t * s.t + c, n);
  }
};
// ... and of B and C.
template <typename T, int SL>
struct Coefs {
  static constexpr int K = kRun * Wave<SL>::NP / 64 > 0 ? kRun * Wave<SL>::NP / 64 : 1;
  T b[K], c[K];
  __device__ __forceinline__ void load(const SelArgs& p, const At& at, int t0, int lane) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = lane + 64 * k, t = t0 + i / Wave<SL>::NP, n = i % Wave<SL>::NP;
      b[k] = c[k] = (T)0.0f;
      if (i < kRun * Wave<SL>::NP && t < at.len && n < p.N) {
        b[k] = static_cast<const T*>(p.B.p)[at.b * p.B.b + (int64_t)t * p.B.t + n];
        c[k] = static_cast<const T*>(p.C.p)[at.b * p.C.b + (int64_t)t * p.C.t + n];
      }
    }
  }
  __device__ __forceinline__ void put(WaveLds<SL>& lds, int lane) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = lane + 64 * k, r = i / Wave<SL>::NP, n = i % Wave<SL>::NP;
      if (i < kRun * Wave<SL>::NP) {
        lds.bc[r][0][n / 4].v[n % 4] = (float)b[k];
        lds.bc[r][1][n / 4].v[n % 4] = (float)c[k];
      }
    }
  }
};

// ---- forward ------------------------------------------------------------------------------------

enum Mode { kWhole, kMaps };

// A workgroup carries a group of channels through a segment of time, a tile of four waves by eight steps at a time.  MAPS:
// only the segment's map is wanted.
template <typename T, int SL, Mode MODE>
__global__ void __launch_bounds__(kWaves* kWave) selective_forward_kernel(SelArgs p) {
  using W = Wave<SL>;
  constexpr int E = W::E;
  __shared__ WaveLds<SL> lds_all[kWaves];
  __shared__ MapLds maps[2][kWaves][2];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  WaveLds<SL>& lds = lds_all[wave];
  const int seg = blockIdx.y;
  const At at = place(p, slab_of(blockIdx.x, gridDim.x), W::CH);
  const Slots<SL> mine(p, at, lane);
  const int64_t state_size = p.batch * p.D_ * p.N;

  // the layout that memory is read and written in
  const int row = lane / 8, ec = lane % 8 * E, c = at.c0 + ec, n = min(max(p.D_ - c, 0), E);
  float bias[E], skip[E], A[kSlots];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    bias[j] = j < n ? param<T>(p.bias, p.w32, c + j, 0.0f) : 0.0f;
    skip[j] = j < n ? param<T>(p.D, p.w32, c + j, 0.0f) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int s = mine.n + i % kNs;
    A[i] = i / kNs < mine.channels && s < p.N
               ? kOpLog2e * param<T>(p.A, p.w32, (int64_t)(mine.c + i / kNs) * p.N + s, 0.0f) : 0.0f;
  }

  const int live = (at.len + kTileSteps - 1) / kTileSteps;  // tiles that the row reaches
  const int first = seg * p.seg_tiles, last = min(first + p.seg_tiles, p.tiles), live_last = min(last, live);
  float carry[kSlots], decay[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) carry[i] = 0.0f, decay[i] = 1.0f;
  if (MODE == kWhole) {
    if (p.h0) mine.load(p, p.h0, at.b, carry);
    for (int s = 0; s < seg; ++s) {  // the segments before this one
      float P[kSlots], Q[kSlots];
      mine.load(p, p.seg + (int64_t)s * 2 * state_size, at.b, P);
      mine.load(p, p.seg + (int64_t)(s * 2 + 1) * state_size, at.b, Q);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) carry[i] = fmaf(P[i], carry[i], Q[i]);
    }
  }

  Rows<T, SL> nu, nd, nz;
  Coefs<T, SL> nc;
  const auto load = [&](int tile) __attribute__((always_inline)) {
    const int t0 = tile * kTileSteps + wave * kRun, t = t0 + row;
    nu.load(p.u, at, t, c, n);
    nd.load(p.dt, at, t, c, n);
    if (MODE == kWhole && p.z.p) nz.load(p.z, at, t, c, n);
    nc.load(p, at, t0, lane);
  };
  nz.v = {};
  if (first < live_last) load(first);
  for (int tile = first; tile < live_last; ++tile) {
    const int t = tile * kTileSteps + wave * kRun + row;
    // dt and dt u, B, C: into the wave's LDS
    Vec<T, E> u = nu.v, z = nz.v;
    {
      float f[2 * E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float raw = (float)nd.v.v[j] + bias[j], dt = t < at.len ? p.softplus ? softplus_of(raw) : raw : 0.0f;
        f[2 * j] = dt, f[2 * j + 1] = dt * (float)u.v[j];
      }
      float* const dst = &lds.step[row][0].v[0] + 2 * ec;
      __builtin_memcpy(__builtin_assume_aligned(dst, 2 * E * 4 < 16 ? 8 : 16), f, sizeof(f));
      nc.put(lds, lane);
    }
    if (tile + 1 < live_last) load(tile + 1);
    wave_sync();
    // 1. decays and the run's map
    float a[kRun][kSlots], Q[kSlots], sum[kCh] = {};
#pragma unroll
    for (int i = 0; i < kSlots; ++i) Q[i] = 0.0f;
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
      const F4 s = lds.step[r][lane / SL], B = lds.bc[r][0][lane % SL];
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        a[r][i] = __builtin_amdgcn_exp2f(s.v[i / kNs * 2] * A[i]);
        Q[i] = fmaf(a[r][i], Q[i], s.v[i / kNs * 2 + 1] * B.v[i % kNs]);
      }
      sum[0] += s.v[0], sum[1] += s.v[2];
    }
    // 2. the waves' maps
    float P[kSlots], h[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) P[i] = run_decay(sum[i / kNs] * A[i]);
    MapLds(*const map)[2] = maps[tile & 1];
    put_map(map[wave][0], lane, P);
    put_map(map[wave][1], lane, Q);
    if (MODE == kWhole && p.states && wave == 0) mine.store(p, p.states + tile * state_size, at.b, carry);
    lds_barrier();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) {
#pragma unroll
        for (int i = 0; i < kSlots; ++i) h[i] = carry[i];
      }
      get_map(map[w][0], lane, P);
      get_map(map[w][1], lane, Q);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        carry[i] = fmaf(P[i], carry[i], Q[i]);
        if (MODE == kMaps) decay[i] = fmaxf(decay[i] * P[i], 0x1p-126f);
      }
    }
    if (MODE == kMaps) continue;
    // 3. the steps from where they start
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
      const F4 s = lds.step[r][lane / SL], B = lds.bc[r][0][lane % SL], C = lds.bc[r][1][lane % SL];
      float y[kCh] = {};
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        h[i] = fmaf(a[r][i], h[i], s.v[i / kNs * 2 + 1] * B.v[i % kNs]);
        y[i / kNs] = fmaf(C.v[i % kNs], h[i], y[i / kNs]);
      }
#pragma unroll
      for (int i = 0; i < kCh; ++i) y[i] = states_sum<SL>(y[i]);
      if (lane % SL == 0) *reinterpret_cast<F2*>(&lds.y[r][lane / SL * kCh]) = F2{{y[0], y[1]}};
    }
    wave_sync();
    if (t < p.T_ && n > 0) {
      float y[E];
      __builtin_memcpy(y, __builtin_assume_aligned(&lds.y[row][ec], E * 4 < 16 ? E * 4 : 16), sizeof(y));
#pragma unroll
      for (int j = 0; j < E; ++j) {
        y[j] = fmaf(skip[j], (float)u.v[j], y[j]);
        if (p.z.p) y[j] *= silu((float)z.v[j]);
        if (t >= at.len) y[j] = 0.0f;
      }
      store_some<T, E>(static_cast<T*>(p.out) + (at.b * p.T_ + t) * p.D_ + c, round_to<T, E>(y), n);
    }
    wave_sync();
  }
  if (MODE == kMaps) {
    if (wave == 0) {
      mine.store(p, p.seg + (int64_t)seg * 2 * state_size, at.b, decay);
      mine.store(p, p.seg + (int64_t)(seg * 2 + 1) * state_size, at.b, carry);
    }
    return;
  }
  for (int tile = max(first, live); tile < last; ++tile) {  // past the row
    const int t = tile * kTileSteps + wave * kRun + row;
    if (t < p.T_ && n > 0) store_some<T, E>(static_cast<T*>(p.out) + (at.b * p.T_ + t) * p.D_ + c, Vec<T, E>{}, n);
  }
  // (the last segment's carry is the row's: past the row nothing changes it)
  if (p.h_n && wave == 0 && seg == p.segs - 1) mine.store(p, p.h_n, at.b, carry);
}

// ---- one token ----------------------------------------------------------------------------------

// SL threads per channel with four states each, for ROWS rows one after the other with the channel's decays in registers.
template <typename T, int SL, int ROWS>
__global__ void __launch_bounds__(256) selective_step_kernel(SelArgs p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, at = i / SL, rows = at / (uint32_t)p.D_;  // (less than 2^32 threads)
  const int d = (int)(at % (uint32_t)p.D_), n0 = (int)(i % SL) * kNs, n = p.N - n0;
  if ((int64_t)rows * ROWS >= p.batch) return;  // (whole groups of SL lanes)
  float A[kNs];
#pragma unroll
  for (int j = 0; j < kNs; ++j) A[j] = j < n ? kOpLog2e * param<T>(p.A, p.w32, (int64_t)d * p.N + n0 + j, 0.0f) : 0.0f;
  const float bias = param<T>(p.bias, p.w32, d, 0.0f), skip = param<T>(p.D, p.w32, d, 0.0f);
  Vec<float, kNs> h[ROWS];
  Vec<T, kNs> B[ROWS], C[ROWS];
  T u[ROWS], raw[ROWS], z[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t b = (int64_t)rows * ROWS + r;
    h[r] = {}, B[r] = {}, C[r] = {};
    u[r] = raw[r] = z[r] = (T)0.0f;
    if (b >= p.batch) continue;
    u[r] = static_cast<const T*>(p.u.p)[b * p.u.b + d];
    raw[r] = static_cast<const T*>(p.dt.p)[b * p.dt.b + d];
    if (p.z.p) z[r] = static_cast<const T*>(p.z.p)[b * p.z.b + d];
    if (n <= 0) continue;
    h[r] = load_some<float, kNs>(p.h0 + (b * p.D_ + d) * p.N + n0, n);
    B[r] = load_some<T, kNs>(static_cast<const T*>(p.B.p) + b * p.B.b + n0, n);
    C[r] = load_some<T, kNs>(static_cast<const T*>(p.C.p) + b * p.C.b + n0, n);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t b = (int64_t)rows * ROWS + r;
    const float v = (float)raw[r] + bias, dt = p.softplus ? softplus_of(v) : v, du = dt * (float)u[r];
    float y = 0.0f;
#pragma unroll
    for (int j = 0; j < kNs; ++j) {
      h[r].v[j] = fmaf(__builtin_amdgcn_exp2f(dt * A[j]), h[r].v[j], du * (float)B[r].v[j]);
      if (j < n) y = fmaf((float)C[r].v[j], h[r].v[j], y);
    }
    y = fmaf(skip, (float)u[r], states_sum<SL>(y));
    if (p.z.p) y *= silu((float)z[r]);
    if (b >= p.batch) continue;
    if (n > 0) store_some<float, kNs>(p.h_n + (b * p.D_ + d) * p.N + n0, h[r], n);
    if (i % SL == 0) static_cast<T*>(p.out)[b * p.D_ + d] = round_to<T>(y);
  }
}

// ---- backward -----------------------------------------------------------------------------------

constexpr int kSide = 2;  // groups of channels of a workgroup, whose dB and dC it adds up

template <int SL>
struct BackLds {
  WaveLds<SL> f;                    // (y: dy, then y; step: then s1, s2 of the pair's two channels)
  float bc[kRun][2][Wave<SL>::NP];  // dB and dC of the wave's channels
};

// The tiles of a segment from the last to the first.  MAPS: only the segment's map of E is wanted.
template <typename T, int SL, Mode MODE>
__global__ void __launch_bounds__(kSide* kWaves* kWave) selective_backward_kernel(SelArgs p) {
  using W = Wave<SL>;
  constexpr int E = W::E;
  __shared__ BackLds<SL> lds_all[kSide][kWaves];
  __shared__ MapLds maps[kSide][kWaves][3];
  const int lane = threadIdx.x % kWave, id = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wave = id % kWaves, side = id / kWaves;
  BackLds<SL>& back = lds_all[side][wave];
  WaveLds<SL>& lds = back.f;
  const int seg = blockIdx.y;
  const int64_t slab = slab_of(blockIdx.x, gridDim.x);
  // A row's groups are taken in pairs (the last one may be alone); rows of one group each, in pairs of rows.
  const bool pair_rows = p.groups == 1;
  const int per_row = (p.groups + kSide - 1) / kSide;
  const int64_t b_of = pair_rows ? slab * kSide + side : slab / per_row;
  const int group = pair_rows ? 0 : (int)(slab % per_row) * kSide + side;
  const bool on = b_of < p.batch && group < p.groups;
  const At at = place(p, on ? b_of * p.groups + group : p.units, W::CH);
  const Slots<SL> mine(p, at, lane);
  const int64_t state_size = p.batch * p.D_ * p.N;

  const int row = lane / 8, ec = lane % 8 * E, c = at.c0 + ec, n = min(max(p.D_ - c, 0), E);
  float bias[E], skip[E], A[kSlots];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    bias[j] = j < n ? param<T>(p.bias, p.w32, c + j, 0.0f) : 0.0f;
    skip[j] = j < n ? param<T>(p.D, p.w32, c + j, 0.0f) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int s = mine.n + i % kNs;
    A[i] = i / kNs < mine.channels && s < p.N
               ? kOpLog2e * param<T>(p.A, p.w32, (int64_t)(mine.c + i / kNs) * p.N + s, 0.0f) : 0.0f;
  }

  const auto length = [&](int64_t b) { return b >= p.batch ? 0 : p.lengths ? min(max(p.lengths[b], 0), p.T_) : p.T_; };
  const int row_len = length(b_of);  // (also of a wave without a group: it adds up its row's dB and dC)
  const int most = pair_rows ? max(row_len, length(slab * kSide + 1 - side)) : row_len;  // the same in all waves
  const int live = (most + kTileSteps - 1) / kTileSteps;
  const int first = seg * p.seg_tiles, last = min(first + p.seg_tiles, p.tiles), live_last = min(last, live);
  float carry[kSlots], decay[kSlots], dA[kSlots], d_skip[E], d_bias[E];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) carry[i] = dA[i] = 0.0f, decay[i] = 1.0f;
#pragma unroll
  for (int j = 0; j < E; ++j) d_skip[j] = d_bias[j] = 0.0f;
  if (MODE == kWhole) {
    if (p.d_hn) mine.load(p, p.d_hn, at.b, carry);
    for (int s = p.segs - 1; s > seg; --s) {  // the segments after this one
      float P[kSlots], Q[kSlots];
      mine.load(p, p.seg + (int64_t)s * 2 * state_size, at.b, P);
      mine.load(p, p.seg + (int64_t)(s * 2 + 1) * state_size, at.b, Q);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) carry[i] = fmaf(P[i], carry[i], Q[i]);
    }
  }

  const Strided d_out = {p.d_out, (int64_t)p.T_ * p.D_, p.D_};
  Rows<T, SL> nu, nd, nz, ng;
  Coefs<T, SL> nc;
  float nh[kSlots];
  const auto load = [&](int tile) __attribute__((always_inline)) {
    const int t0 = tile * kTileSteps + wave * kRun, t = t0 + row;
    ng.load(d_out, at, t, c, n);
    nd.load(p.dt, at, t, c, n);
    if (MODE == kWhole) nu.load(p.u, at, t, c, n);
    if (p.z.p) nz.load(p.z, at, t, c, n);
    nc.load(p, at, t0, lane);
    if (MODE == kWhole) {
#pragma unroll
      for (int i = 0; i < kSlots; ++i) nh[i] = 0.0f;
      if (tile * kTileSteps < at.len) mine.load(p, p.states + tile * state_size, at.b, nh);
    }
  };
  nz.v = {}, nu.v = {};
  // dB and dC of a tile that is done (its waves have met at a barrier since)
  const int64_t bc_group = pair_rows ? 0 : slab % per_row;
  const auto flush = [&](int tile) __attribute__((always_inline)) {
    const int t0 = tile * kTileSteps + wave * kRun;
    for (int i = (pair_rows ? 0 : side * kWave) + lane; i < kRun * 2 * W::NP; i += (pair_rows ? 1 : kSide) * kWave) {
      const int r = i / (2 * W::NP), k = i / W::NP % 2, s = i % W::NP, t = t0 + r;
      if (t >= row_len || s >= p.N) continue;
      float v = lds_all[pair_rows ? side : 0][wave].bc[r][k][s];
      if (!pair_rows) v += lds_all[1][wave].bc[r][k][s];
      p.part_bc[((bc_group * p.batch + b_of) * p.T_ + t) * 2 * p.N + k * p.N + s] = v;
    }
  };
  if (first < live_last) load(live_last - 1);
  for (int tile = live_last - 1; tile >= first; --tile) {
    const int t = tile * kTileSteps + wave * kRun + row;
    const Vec<T, E> u = nu.v, z = nz.v, g = ng.v, d = nd.v;
    float dt[E], dy[E], start[kSlots];
    {
      float f[2 * E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float raw = (float)d.v[j] + bias[j];
        dt[j] = t < at.len ? p.softplus ? softplus_of(raw) : raw : 0.0f;
        f[2 * j] = dt[j], f[2 * j + 1] = dt[j] * (float)u.v[j];
        dy[j] = (float)g.v[j];
        if (p.z.p) dy[j] *= silu((float)z.v[j]);
      }
      float* const dst = &lds.step[row][0].v[0] + 2 * ec;
      __builtin_memcpy(__builtin_assume_aligned(dst, 2 * E * 4 < 16 ? 8 : 16), f, sizeof(f));
      __builtin_memcpy(__builtin_assume_aligned(&lds.y[row][ec], E * 4 < 16 ? E * 4 : 16), dy, sizeof(dy));
      nc.put(lds, lane);
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) start[i] = nh[i];
    if (tile > first) load(tile - 1);
    wave_sync();
    // 1. decays, the run's maps forward (h) and backward (E)
    float a[kRun][kSlots], Qh[kSlots], Qe[kSlots], sum[kCh] = {};
#pragma unroll
    for (int i = 0; i < kSlots; ++i) Qh[i] = Qe[i] = 0.0f;
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
      const F4 s = lds.step[r][lane / SL], B = lds.bc[r][0][lane % SL];
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        a[r][i] = __builtin_amdgcn_exp2f(s.v[i / kNs * 2] * A[i]);
        if (MODE == kWhole) Qh[i] = fmaf(a[r][i], Qh[i], s.v[i / kNs * 2 + 1] * B.v[i % kNs]);
      }
      sum[0] += s.v[0], sum[1] += s.v[2];
    }
#pragma unroll
    for (int r = kRun - 1; r >= 0; --r) {
      const F4 C = lds.bc[r][1][lane % SL];
      const F2 q = *reinterpret_cast<const F2*>(&lds.y[r][lane / SL * kCh]);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) Qe[i] = a[r][i] * fmaf(C.v[i % kNs], q.v[i / kNs], Qe[i]);
    }
    // 2. the waves' maps
    float P[kSlots], h[kSlots], e[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) P[i] = run_decay(sum[i / kNs] * A[i]);
    MapLds(*const map)[3] = maps[side];
    put_map(map[wave][0], lane, P);
    put_map(map[wave][1], lane, Qe);
    if (MODE == kWhole) put_map(map[wave][2], lane, Qh);
    lds_barrier();
    if (MODE == kWhole && tile + 1 < live_last) flush(tile + 1);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) h[i] = start[i];
#pragma unroll
    for (int w = kWaves - 1; w >= 0; --w) {
      if (w == wave) {
#pragma unroll
        for (int i = 0; i < kSlots; ++i) e[i] = carry[i];
      }
      get_map(map[w][0], lane, P);
      get_map(map[w][1], lane, Qe);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        carry[i] = fmaf(P[i], carry[i], Qe[i]);
        if (MODE == kMaps) decay[i] = fmaxf(decay[i] * P[i], 0x1p-126f);
      }
    }
    if (MODE == kWhole) {
#pragma unroll
      for (int w = 0; w + 1 < kWaves; ++w) {
        if (w >= wave) break;
        get_map(map[w][0], lane, P);
        get_map(map[w][2], lane, Qh);
#pragma unroll
        for (int i = 0; i < kSlots; ++i) h[i] = fmaf(P[i], h[i], Qh[i]);
      }
    }
    lds_barrier();  // (the maps and the sums of the tile before have been read)
    if (MODE == kMaps) continue;
    // 3. the states, step by step, each before its step; with a gate the outputs that it multiplies
    float before[kRun][kSlots], out[kRun][kCh];
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
      const F4 s = lds.step[r][lane / SL], B = lds.bc[r][0][lane % SL], C = lds.bc[r][1][lane % SL];
      out[r][0] = out[r][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        before[r][i] = h[i];
        h[i] = fmaf(a[r][i], h[i], s.v[i / kNs * 2 + 1] * B.v[i % kNs]);
        out[r][i / kNs] = fmaf(C.v[i % kNs], h[i], out[r][i / kNs]);
      }
    }
    // 4. and backwards
    const auto walk = [&](auto whole) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
    for (int r = kRun - 1; r >= 0; --r) {
      const F4 s = lds.step[r][lane / SL], B = lds.bc[r][0][lane % SL], C = lds.bc[r][1][lane % SL];
      const F2 q = *reinterpret_cast<const F2*>(&lds.y[r][lane / SL * kCh]);
      const bool in = WHOLE || tile * kTileSteps + wave * kRun + r < at.len;
      float s1[kCh] = {}, s2[kCh] = {}, dB[kNs] = {}, dC[kNs] = {};
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        const int k = i / kNs, j = i % kNs;
        const float G = fmaf(C.v[j], q.v[k], e[i]);
        s1[k] = fmaf(G, B.v[j], s1[k]);
        dB[j] = fmaf(G, s.v[2 * k + 1], dB[j]);
        dC[j] = fmaf(q.v[k], r + 1 < kRun ? before[r + 1 < kRun ? r + 1 : r][i] : h[i], dC[j]);
        e[i] = a[r][i] * G;
        const float m = in ? e[i] * before[r][i] : 0.0f;  // (past the row it may be inf * 0)
        s2[k] = fmaf(m, A[i], s2[k]);
        dA[i] = fmaf(m, s.v[2 * k], dA[i]);
      }
#pragma unroll
      for (int k = 0; k < kCh; ++k) {
        s1[k] = states_sum<SL>(s1[k]);
        s2[k] = states_sum<SL>(s2[k]);
        if (p.z.p) out[r][k] = states_sum<SL>(out[r][k]);
      }
      // dB to the low half, dC to the high one, states 0, 2 to the even rows of 16 lanes, 1, 3 to the odd ones
      float w[kNs], x[2];
#pragma unroll
      for (int j = 0; j < kNs; ++j) w[j] = pair_sum<true>(dB[j], dC[j]);
      x[0] = row_rest_sum<SL>(pair_sum<false>(w[0], w[1]));
      x[1] = row_rest_sum<SL>(pair_sum<false>(w[2], w[3]));
      if (lane % 16 < SL) {
        float* const dst = &back.bc[r][lane / 32][lane % SL * kNs + lane / 16 % 2];
        dst[0] = x[0], dst[2] = x[1];
      }
      if (lane % SL == 0) {
        constexpr float kLn2 = 0.69314718f;
        lds.step[r][lane / SL] = F4{{s1[0], s2[0] * kLn2, s1[1], s2[1] * kLn2}};
        if (p.z.p) *reinterpret_cast<F2*>(&lds.y[r][lane / SL * kCh]) = F2{{out[r][0], out[r][1]}};
      }
    }
    };
    if (tile * kTileSteps + (wave + 1) * kRun <= at.len)
      walk(std::true_type());
    else
      walk(std::false_type());
    wave_sync();
    if (t < p.T_ && n > 0) {
      float f[2 * E], y[E], du[E], dr[E], dz[E];
      __builtin_memcpy(f, __builtin_assume_aligned(&lds.step[row][0].v[0] + 2 * ec, 2 * E * 4 < 16 ? 8 : 16), sizeof(f));
      __builtin_memcpy(y, __builtin_assume_aligned(&lds.y[row][ec], E * 4 < 16 ? E * 4 : 16), sizeof(y));
      const bool in = t < at.len;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float uj = (float)u.v[j];
        du[j] = in ? fmaf(dt[j], f[2 * j], dy[j] * skip[j]) : 0.0f;
        dr[j] = fmaf(uj, f[2 * j], f[2 * j + 1]);
        if (p.softplus) dr[j] *= sigmoid((float)d.v[j] + bias[j]);
        if (!in) dr[j] = 0.0f;
        if (in) d_skip[j] = fmaf(dy[j], uj, d_skip[j]);
        d_bias[j] += dr[j];
        if (p.z.p) {
          const float zj = (float)z.v[j];
          dz[j] = in ? (float)g.v[j] * fmaf(skip[j], uj, y[j]) * silu_slope(zj) : 0.0f;
        }
      }
      const int64_t o = (at.b * p.T_ + t) * p.D_ + c;
      store_some<T, E>(static_cast<T*>(p.d_u) + o, round_to<T, E>(du), n);
      store_some<T, E>(static_cast<T*>(p.d_dt) + o, round_to<T, E>(dr), n);
      if (p.z.p) store_some<T, E>(static_cast<T*>(p.d_z) + o, round_to<T, E>(dz), n);
    }
    wave_sync();
  }
  if (MODE == kMaps) {
    if (wave == 0) {
      mine.store(p, p.seg + (int64_t)seg * 2 * state_size, at.b, decay);
      mine.store(p, p.seg + (int64_t)(seg * 2 + 1) * state_size, at.b, carry);
    }
    return;
  }
  for (int tile = max(first, live_last); tile < last; ++tile) {  // past the row
    const int t = tile * kTileSteps + wave * kRun + row;
    if (t >= p.T_ || n <= 0) continue;
    const int64_t o = (at.b * p.T_ + t) * p.D_ + c;
    store_some<T, E>(static_cast<T*>(p.d_u) + o, Vec<T, E>{}, n);
    store_some<T, E>(static_cast<T*>(p.d_dt) + o, Vec<T, E>{}, n);
    if (p.z.p) store_some<T, E>(static_cast<T*>(p.d_z) + o, Vec<T, E>{}, n);
  }
  if (p.d_h0 && wave == 0 && seg == 0) mine.store(p, p.d_h0, at.b, carry);

  // The waves' sums of dA, dD and dbias, added in their order.
  lds_barrier();
  if (first < live_last) flush(first);
  lds_barrier();
  float* const part = p.part_w + ((int64_t)seg * p.batch + at.b) * p.D_ * (p.N + 2);
  put_map(maps[side][wave][0], lane, dA);
  // (lanes that share a channel: the eight rows)
  float(*const edge)[2 * E] = reinterpret_cast<float(*)[2 * E]>(&back);  // [64]
  wave_sync();
#pragma unroll
  for (int j = 0; j < E; ++j) edge[lane][j] = d_skip[j], edge[lane][E + j] = d_bias[j];
  lds_barrier();
  if (wave == 0) {
    float v[kSlots];
    for (int w = 1; w < kWaves; ++w) {
      get_map(maps[side][w][0], lane, v);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) dA[i] += v[i];
    }
    mine.store(p, part - at.b * p.D_ * p.N, at.b, dA);
  } else if (wave == 1 && lane < 16) {
    // eight lanes with E channels each, for dD and for dbias
    const int k = lane / 8;
    float v[E] = {};
    for (int w = 0; w < kWaves; ++w) {
      const float(*const other)[2 * E] = reinterpret_cast<const float(*)[2 * E]>(&lds_all[side][w]);
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] += other[r * 8 + lane % 8][k * E + j];
    }
    Vec<float, E> out;
#pragma unroll
    for (int j = 0; j < E; ++j) out.v[j] = v[j];
    const int cc = at.c0 + lane % 8 * E;
    if (p.D_ > cc) store_some<float, E>(part + (int64_t)p.D_ * (p.N + k) + cc, out, p.D_ - cc);
  }
}

// dB and dC: the workgroups' sums, in their order.
template <typename T>
__global__ void __launch_bounds__(256) selective_coefs_kernel(SelArgs p, T* d_B, T* d_C) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = p.batch * p.T_;
  if (i >= rows * 2 * p.N) return;
  const int64_t row = i / (2 * p.N), b = row / p.T_;
  const int k = (int)(i % (2 * p.N)), t = (int)(row % p.T_);
  float s = 0.0f;
  if (!p.lengths || t < p.lengths[b]) {
#pragma unroll 8
    for (int g = 0; g < p.bc_groups; ++g) s += p.part_bc[g * rows * 2 * p.N + i];
  }
  T* const dst = k < p.N ? d_B : d_C;
  if (dst) dst[row * p.N + (k < p.N ? k : k - p.N)] = round_to<T>(s);
}

// ---- host ---------------------------------------------------------------------------------------

int state_lanes(int states) {
  int sl = 1;
  while (sl * kNs < states) sl *= 2;
  return sl;
}

struct SelLayout {
  int groups;     // of channels, in a row
  int tiles, seg_tiles, segs;
  int bc_groups;  // sums of dB and dC
};

// Segments of the time axis so that the launch has about `want` workgroups.
SelLayout sel_layout(int64_t batch, int64_t seq_len, int64_t channels, int states, bool backward) {
  SelLayout l;
  const int per = 64 / state_lanes(states) * kCh;
  l.groups = (int)((channels + per - 1) / per);
  l.bc_groups = (l.groups + kSide - 1) / kSide;
  l.tiles = (int)((seq_len + kTileSteps - 1) / kTileSteps);
  l.seg_tiles = std::max(l.tiles, 1);
  l.segs = 1;
  (void)batch, (void)backward;
  return l;
}

struct SelWorkspace {
  int64_t seg, bc, w, bytes;  // offsets in floats; bytes of all
};
SelWorkspace sel_workspace(int64_t batch, int64_t seq_len, int64_t channels, int states, bool backward) {
  const SelLayout l = sel_layout(batch, seq_len, channels, states, backward);
  SelWorkspace s = {};
  const auto round = [](int64_t n) { return (n + 3) / 4 * 4; };
  s.bc = l.segs > 1 ? round((int64_t)l.segs * 2 * batch * channels * states) : 0;
  s.w = s.bc + (backward ? round((int64_t)l.bc_groups * batch * seq_len * 2 * states) : 0);
  s.bytes = 4 * (s.w + (backward ? round((int64_t)l.segs * batch * channels * (states + 2)) : 0));
  return s;
}

// f(std::integral_constant of the lanes).
template <typename F>
hipError_t with_lanes(int states, F&& f) {
  switch (state_lanes(states)) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 4: return f(std::integral_constant<int, 4>());
    case 8: return f(std::integral_constant<int, 8>());
    case 16: return f(std::integral_constant<int, 16>());
    default: return hipErrorInvalidValue;
  }
}

template <typename T>
hipError_t launch_sel_forward(const SelArgs& p, hipStream_t s) {
  return with_lanes(p.N, [&](auto lanes) {
    constexpr int SL = decltype(lanes)::value;
    const dim3 block(kWaves * kWave);
    if (p.segs > 1) {
      hipLaunchKernelGGL((selective_forward_kernel<T, SL, kMaps>), dim3((unsigned)p.units, p.segs - 1), block, 0, s, p);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((selective_forward_kernel<T, SL, kWhole>), dim3((unsigned)p.units, p.segs), block, 0, s, p);
    return hipGetLastError();
  });
}

template <typename T>
hipError_t launch_sel_step(const SelArgs& p, hipStream_t s) {
  return with_lanes(p.N, [&](auto lanes) {
    constexpr int SL = decltype(lanes)::value;
    const auto run = [&](auto rows) {
      constexpr int ROWS = decltype(rows)::value;
      const dim3 grid((unsigned)(((p.batch + ROWS - 1) / ROWS * p.D_ * SL + 255) / 256));
      hipLaunchKernelGGL((selective_step_kernel<T, SL, ROWS>), grid, dim3(256), 0, s, p);
      return hipGetLastError();
    };
    return p.batch * p.D_ * SL >= 4 * 256 * 1024 ? run(std::integral_constant<int, 4>()) : run(std::integral_constant<int, 1>());
  });
}

template <typename T>
hipError_t launch_sel_backward(SelArgs p, void* d_A, void* d_B, void* d_C, void* d_D, void* d_bias, hipStream_t s) {
  hipError_t e = hipSuccess;
  if (p.batch > 0) {
    const int64_t slabs = p.groups == 1 ? (p.batch + kSide - 1) / kSide : p.batch * ((p.groups + kSide - 1) / kSide);
    e = with_lanes(p.N, [&](auto lanes) {
      constexpr int SL = decltype(lanes)::value;
      const dim3 block(kSide * kWaves * kWave);
      if (p.segs > 1) {
        hipLaunchKernelGGL((selective_backward_kernel<T, SL, kMaps>), dim3((unsigned)slabs, p.segs), block, 0, s, p);
        const hipError_t e2 = hipGetLastError();
        if (e2 != hipSuccess) return e2;
      }
      hipLaunchKernelGGL((selective_backward_kernel<T, SL, kWhole>), dim3((unsigned)slabs, p.segs), block, 0, s, p);
      return hipGetLastError();
    });
    const int64_t n = p.batch * p.T_ * 2 * p.N;
    if (e == hipSuccess && n > 0 && (d_B || d_C)) {
      hipLaunchKernelGGL(selective_coefs_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, (T*)d_B, (T*)d_C);
      e = hipGetLastError();
    }
  }
  if (e == hipSuccess && (d_A || d_D || d_bias)) {
    ColumnSums sums = {};
    sums.part = p.part_w, sums.rows = (int64_t)p.segs * p.batch, sums.cols = (int64_t)p.D_ * (p.N + 2), sums.out32 = p.w32;
    sums.out[0] = d_A, sums.out[1] = d_D, sums.out[2] = d_bias;
    sums.begin[1] = (int64_t)p.D_ * p.N, sums.begin[2] = sums.begin[1] + p.D_, sums.begin[3] = sums.cols;
    e = launch_column_sums<T>(sums, s);
  }
  return e;
}

int check_selective(const char* what, const plh_selective_scan_args* a) noexcept {
  if (!a) return op_error(PLH_ERR_INVALID, what, "args is required");
  if (a->dtype != PLH_F16 && a->dtype != PLH_BF16 && a->dtype != PLH_F32)
    return op_error(PLH_ERR_INVALID, what, "dtype must be PLH_F16, PLH_BF16 or PLH_F32");
  if (a->wdtype != a->dtype && a->wdtype != PLH_F32)
    return op_error(PLH_ERR_INVALID, what, "wdtype must be dtype or PLH_F32");
  if (a->batch < 0 || a->seq_len < 0) return op_error(PLH_ERR_INVALID, what, "batch and seq_len must be non-negative");
  if (a->states < 1 || a->states > kMaxStates) return op_error(PLH_ERR_UNSUPPORTED, what, "states must lie in [1, 64]");
  if (a->channels < 1 || a->channels > (1 << 24))
    return op_error(PLH_ERR_UNSUPPORTED, what, "channels must lie in [1, 2^24]");
  if (a->seq_len > (1 << 30)) return op_error(PLH_ERR_UNSUPPORTED, what, "seq_len must not exceed 2^30");
  if (a->batch > (1 << 23) || a->batch * ((a->channels + 7) / 8) > (1 << 23))
    return op_error(PLH_ERR_UNSUPPORTED, what, "batch * ceil(channels / 8) must not exceed 2^23");
  if (a->batch * a->seq_len * a->states > (1 << 30))
    return op_error(PLH_ERR_UNSUPPORTED, what, "batch * seq_len * states must not exceed 2^30");
  if (!a->A) return op_error(PLH_ERR_INVALID, what, "A is required");
  if (a->batch > 0 && a->seq_len > 0 && (!a->u || !a->dt || !a->B || !a->C))
    return op_error(PLH_ERR_INVALID, what, "u, dt, B and C are required");
  for (const int64_t* st : {a->u_stride, a->dt_stride, a->z_stride, a->B_stride, a->C_stride})
    if (st[0] < 0 || st[1] < 0) return op_error(PLH_ERR_INVALID, what, "strides must be non-negative");
  return PLH_OK;
}

SelArgs sel_args(const plh_selective_scan_args* a, bool backward) {
  SelArgs p = {};
  p.u = {a->u, a->u_stride[0], a->u_stride[1]}, p.dt = {a->dt, a->dt_stride[0], a->dt_stride[1]};
  p.z = {a->z, a->z_stride[0], a->z_stride[1]};
  p.B = {a->B, a->B_stride[0], a->B_stride[1]}, p.C = {a->C, a->C_stride[0], a->C_stride[1]};
  p.A = a->A, p.D = a->D, p.bias = a->dt_bias, p.w32 = a->wdtype == PLH_F32, p.softplus = a->softplus != 0;
  p.lengths = a->lengths, p.batch = a->batch, p.T_ = (int)a->seq_len, p.D_ = (int)a->channels, p.N = a->states;
  const SelLayout l = sel_layout(a->batch, a->seq_len, a->channels, a->states, backward);
  p.groups = l.groups, p.units = a->batch * l.groups, p.tiles = l.tiles, p.seg_tiles = l.seg_tiles, p.segs = l.segs;
  p.bc_groups = l.bc_groups;
  return p;
}

}  // namespace
}  // namespace plh

extern "C" {

int64_t plh_selective_scan_states(int64_t seq_len) {
  return seq_len < 0 ? -1 : (seq_len + plh::kTileSteps - 1) / plh::kTileSteps;
}

int64_t plh_selective_scan_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int states, int backward) {
  if (batch < 0 || seq_len < 0 || seq_len > (1 << 30) || channels < 1 || channels > (1 << 24) || states < 1 ||
      states > plh::kMaxStates)
    return -1;
  return plh::sel_workspace(batch, seq_len, channels, states, backward != 0).bytes;
}

int plh_selective_scan_forward(const plh_selective_scan_args* a, const float* h0, void* out, float* h_n, float* states,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* const what = "selective_scan_forward";
  const int rc = plh::check_selective(what, a);
  if (rc != PLH_OK) return rc;
  if (a->batch == 0) return PLH_OK;
  if (a->seq_len > 0 && !out) return plh::op_error(PLH_ERR_INVALID, what, "out is required");
  const plh::SelWorkspace w = plh::sel_workspace(a->batch, a->seq_len, a->channels, a->states, false);
  if (w.bytes > 0 && (!workspace || workspace_bytes < w.bytes || !plh::aligned(workspace, 16)))
    return plh::op_error(PLH_ERR_INVALID, what,
                         "workspace missing, smaller than plh_selective_scan_workspace_bytes() or not 16-byte aligned");
  plh::SelArgs p = plh::sel_args(a, false);
  p.h0 = h0, p.out = out, p.h_n = h_n, p.states = states, p.seg = (float*)workspace;
  hipError_t e = hipSuccess;
  plh::with_dtype(a->dtype, [&](auto zero) { e = plh::launch_sel_forward<decltype(zero)>(p, (hipStream_t)stream); });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

int plh_selective_scan_step(const plh_selective_scan_args* a, const float* h, void* out, float* h_n, void* stream) {
  const char* const what = "selective_scan_step";
  const int rc = plh::check_selective(what, a);
  if (rc != PLH_OK) return rc;
  if (a->seq_len != 1) return plh::op_error(PLH_ERR_INVALID, what, "seq_len must be 1");
  if (a->lengths) return plh::op_error(PLH_ERR_INVALID, what, "a step has no lengths");
  if (a->batch == 0) return PLH_OK;
  if (!h || !out || !h_n) return plh::op_error(PLH_ERR_INVALID, what, "h, out and h_n are required");
  plh::SelArgs p = plh::sel_args(a, false);
  p.h0 = h, p.out = out, p.h_n = h_n;
  hipError_t e = hipSuccess;
  plh::with_dtype(a->dtype, [&](auto zero) { e = plh::launch_sel_step<decltype(zero)>(p, (hipStream_t)stream); });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

int plh_selective_scan_backward(const plh_selective_scan_args* a, const float* states, const void* d_out,
                                const float* d_hn, const plh_selective_scan_grads* g, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  const char* const what = "selective_scan_backward";
  const int rc = plh::check_selective(what, a);
  if (rc != PLH_OK) return rc;
  if (!g) return plh::op_error(PLH_ERR_INVALID, what, "grads is required");
  if (a->batch > 0 && a->seq_len > 0 && (!states || !d_out || !g->d_u || !g->d_dt || (a->z && !g->d_z)))
    return plh::op_error(PLH_ERR_INVALID, what, "states, d_out, d_u, d_dt and (with z) d_z are required");
  const plh::SelWorkspace w = plh::sel_workspace(a->batch, a->seq_len, a->channels, a->states, true);
  if (w.bytes > 0 && (!workspace || workspace_bytes < w.bytes || !plh::aligned(workspace, 16)))
    return plh::op_error(PLH_ERR_INVALID, what,
                         "workspace missing, smaller than plh_selective_scan_workspace_bytes() or not 16-byte aligned");
  plh::SelArgs p = plh::sel_args(a, true);
  float* const ws = (float*)workspace;
  p.states = const_cast<float*>(states), p.d_out = d_out, p.d_hn = d_hn, p.d_h0 = g->d_h0;
  p.d_u = g->d_u, p.d_dt = g->d_dt, p.d_z = g->d_z;
  p.seg = ws, p.part_bc = ws + w.bc, p.part_w = ws + w.w;
  hipError_t e = hipSuccess;
  plh::with_dtype(a->dtype, [&](auto zero) {
    e = plh::launch_sel_backward<decltype(zero)>(p, g->d_A, g->d_B, g->d_C, g->d_D, g->d_dt_bias, (hipStream_t)stream);
  });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

}  // extern "C"
