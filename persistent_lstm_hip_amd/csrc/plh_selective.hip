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
// backward.  With 16 states the arithmetic takes longer than the traffic, so the layout saves operations.  A thread has
// up to four neighbouring states of a channel for eight consecutive steps, whose decays stay in registers between the passes
// over them:
//   1. the decays, and the map of the thread's eight steps
//   2. the waves of a workgroup are consecutive in time; their maps meet in LDS around one barrier, and every wave folds
//      those before it into its own start
//   3. the eight steps from there, with the outputs
// so that an exponential is taken once although four times as many waves run as there are channels for.  (Two channels
// by four states per thread read B and C half as often, and add up dB and dC in half the operations, but take twice the
// registers: 8 x 2048 x 2048 channels x 16 states bf16 forward 256 -> 320 us, backward 886 -> 1770, with spills; measured
// before the backward pass kept part of its values in LDS.)
// At these sizes the forward kernel now takes 250 us, VALU busy 74% of the time, the backward one 605, 74%, and its sums 62.
// Per state and step it issues 12 instructions forward, of which 5 are the formulas' and 2 those of them that two passes do
// (the input's product and the recurrence); 30 backward, of which 13 and 4.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "plh_ops.h"

namespace plh {
namespace {

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

// A wave's layout: SL threads side by side have the states of a channel, NS neighbouring ones each; 64 / SL channels make
// the wave's group.
template <int SL_, int NS_>
struct Geo {
  static constexpr int SL = SL_, NS = NS_;
  static constexpr int GROUP = 64 / SL, NP = SL * NS;  // NP: states, padded
  // How the wave reads its eight steps of GROUP channels and of NP states: eight lanes per step, with E neighbouring
  // channels and F neighbouring states each.
  static constexpr int E = GROUP >= 8 ? GROUP / 8 : 1, F = NP >= 8 ? NP / 8 : 1;
  static_assert(kRun == 8, "eight steps by eight lanes");
  // Groups of a workgroup of the backward pass, whose dB and dC it adds up.  One leaves three workgroups per CU, with rows
  // of their own pace, two save half of the partial sums' traffic, which grows with the states.  One and two, us of a
  // training call less those of a forward one: 16 states 8 x 2048 x 2048 bf16 650 and 742, 128 x 1000 x 256 fp16 ragged 431
  // and 580; 32 states 4 x 2048 x 1024 bf16 455 and 404, 64 states 1073 and 960.
  static constexpr int SIDE = SL == 4 ? 1 : 2;
};

// Orders the LDS accesses of a wave's lanes among each other (they run in order; this is for the compiler).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

// N floats that are moved at once, in LDS.
template <int N>
struct alignas(N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4) Fs {
  float v[N];
};

template <int N>
using FVec = Vec<float, N>;

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

// softplus(v) = log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|), with log1p(e) = 2 artanh(s), s = e / (2 + e) in
// [0, 1/3]: the logarithm of a number close to one would lose the small values, which step sizes are.  artanh(s) / s is a
// polynomial of degree 4 in s^2, fitted over that range to a relative error of 2^-26.9 at most.  Its slope is sigmoid(v).
__device__ __forceinline__ float log1p_of(float e) {
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
  float t = fmaf(0.140891671f, q, 0.139803007f);
  t = fmaf(t, q, 0.200124547f);
  t = fmaf(t, q, 0.333331585f);
  return 2.0f * fmaf(t * q, s, s);
}
__device__ __forceinline__ float softplus(float v) {
  const float e = __builtin_amdgcn_exp2f(-__builtin_fabsf(v) * kOpLog2e);
  return log1p_of(e) + __builtin_elementwise_maximum(v, 0.0f);
}
__device__ __forceinline__ void softplus(float v, float& value, float& slope) {
  const float e = __builtin_amdgcn_exp2f(-__builtin_fabsf(v) * kOpLog2e), r = __builtin_amdgcn_rcpf(1.0f + e);
  value = log1p_of(e) + __builtin_elementwise_maximum(v, 0.0f);
  slope = v < 0.0f ? e * r : r;
}

// A decay's rate, times log2 e.  Minus infinity becomes the largest finite one: a step of size zero, as past a row's end,
// leaves the state as it is, and 0 * inf would not.
__device__ __forceinline__ float rate(float A) { return __builtin_elementwise_maximum(A * kOpLog2e, -3e38f); }

// The map of a run of steps, h -> P h + Q, with P = 2^log2_decay.  Every step's own decay is positive, but their product may
// be too small for fp32 (or, where step sizes are negative and the state grows, too large), and 0 * inf would be NaN where the
// steps one after the other are not.  So P is held at 2^-126 at least, which leaves next to nothing of a state.  Where it may grow
// again, which it cannot with softplus, P is held as its square root (GROWS), which is in range down to P = 2^-252 and up to
// 2^254: what lies beyond leaves no normal number of a normal one.  (8 x 2048 x 2048 channels x 16 states bf16 forward 236 us,
// backward 667, with the root 240 and 673.)
__device__ __forceinline__ float bounded_exp2(float v) {
  return __builtin_amdgcn_exp2f(__builtin_amdgcn_fmed3f(v, -126.0f, 127.0f));
}
template <bool GROWS>
__device__ __forceinline__ float run_decay(float log2_decay) {
  return bounded_exp2(GROWS ? 0.5f * log2_decay : log2_decay);
}
template <bool GROWS>
__device__ __forceinline__ float apply_map(float P, float Q, float h) {
  return GROWS ? fmaf(P * h, P, Q) : fmaf(P, h, Q);
}

// Waits for what v was loaded from.  (The compiler would wait in the loop that uses v next, every time, and so for that loop's
// own loads too: 8 x 2048 x 2048 channels x 16 states bf16 forward 246 us, with the wait in front of it 235.)
template <int N>
__device__ __forceinline__ void arrived(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

__device__ __forceinline__ bool any_lane(bool v) { return __builtin_amdgcn_ballot_w64(v) != 0; }

// Sum over the SL lanes that share a channel, to all of them.
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
template <typename G>
struct alignas(16) WaveLds {
  Fs<2> step[kRun][G::GROUP];   // dt and dt u of every channel
  Fs<G::NS> bc[kRun][2][G::SL];  // B and C
  float y[kRun][G::GROUP];
};
// A map's factors or sums, of all threads of a wave.
template <typename G>
struct MapLds {
  Fs<G::NS> v[64];
  __device__ __forceinline__ void put(int lane, const float (&f)[G::NS]) {
    Fs<G::NS> t;
#pragma unroll
    for (int j = 0; j < G::NS; ++j) t.v[j] = f[j];
    v[lane] = t;
  }
  __device__ __forceinline__ void get(int lane, float (&f)[G::NS]) const {
    const Fs<G::NS> t = v[lane];
#pragma unroll
    for (int j = 0; j < G::NS; ++j) f[j] = t.v[j];
  }
};

// A thread's states, in [B][D][N] at row b; zero outside.  PADDED: there are fewer states than NP.  Those that are missing have
// B = C = 0 and the smallest rate, which leaves their h and E zero as long as u, dt and dy are finite; an infinity times zero
// would be a NaN in the sums over a channel's states.
template <typename G, bool PADDED>
struct Slots {
  int c, n;    // channel and first state
  int states;  // of the NS that there are
  __device__ __forceinline__ Slots(const SelArgs& p, const At& at, int lane) {
    c = at.c0 + lane / G::SL, n = lane % G::SL * G::NS;
    states = c < p.D_ ? min(max(p.N - n, 0), G::NS) : 0;
  }
  __device__ __forceinline__ void load(const SelArgs& p, const float* base, int64_t b, float (&v)[G::NS]) const {
    const Vec<float, G::NS> t = load_some<float, G::NS>(base + (b * p.D_ + c) * p.N + n, states);
#pragma unroll
    for (int j = 0; j < G::NS; ++j) v[j] = t.v[j];
  }
  __device__ __forceinline__ void store(const SelArgs& p, float* base, int64_t b, const float (&v)[G::NS]) const {
    Vec<float, G::NS> t;
#pragma unroll
    for (int j = 0; j < G::NS; ++j) t.v[j] = v[j];
    store_some<float, G::NS>(base + (b * p.D_ + c) * p.N + n, t, states);
  }
  // v of state i, zero where that is missing.
  __device__ __forceinline__ float of(int i, float v) const { return PADDED && i >= states ? 0.0f : v; }
  __device__ __forceinline__ void clear_missing(float (&v)[G::NS]) const {
#pragma unroll
    for (int i = 0; i < G::NS; ++i) v[i] = of(i, v[i]);
  }
  // The decays' rates, times log2 e.  (Of missing states one that is not zero: an infinite step's decay is then zero, not NaN.)
  template <typename T>
  __device__ __forceinline__ void rates(const SelArgs& p, float (&v)[G::NS]) const {
#pragma unroll
    for (int j = 0; j < G::NS; ++j)
      v[j] = j < states ? rate(param<T>(p.A, p.w32, (int64_t)c * p.N + n + j, 0.0f)) : -0x1p-126f;
  }
};

// A wave's eight steps of a tensor, N elements per lane, as loaded: the lane's place in the tensor, moved from tile to tile.
template <typename T, int N>
struct Rows {
  const T* at;
  int64_t step;
  int n;  // elements that there are
  Vec<T, N> v;
  __device__ __forceinline__ void place(const Strided& s, int64_t b, int64_t t, int c, int count, int steps) {
    at = static_cast<const T*>(s.p) + b * s.b + t * s.t + c, step = s.t * steps, n = count, v = {};
  }
  // The next tile's; nothing where `on` is false.
  __device__ __forceinline__ void load(bool on) {
    v = load_some<T, N>(at, on ? n : 0);
    at += step;
  }
};

// What a wave reads of a tile.
template <typename T, typename G>
struct TileIn {
  Rows<T, G::E> u, dt, z;
  Rows<T, G::F> B, C;
  __device__ __forceinline__ void place(const SelArgs& p, const At& at, int64_t t, int c, int n, int lane, int steps) {
    const int f = lane % 8 * G::F, states = min(max(p.N - f, 0), G::F);
    u.place(p.u, at.b, t, c, n, steps), dt.place(p.dt, at.b, t, c, n, steps);
    if (p.z.p) z.place(p.z, at.b, t, c, n, steps);
    z.v = {};
    B.place(p.B, at.b, t, f, states, steps), C.place(p.C, at.b, t, f, states, steps);
  }
  __device__ __forceinline__ void put_coefs(WaveLds<G>& lds, int lane) const {
    if (G::NP < 8 && lane % 8 >= G::NP) return;
    Fs<G::F> b, c;
#pragma unroll
    for (int j = 0; j < G::F; ++j) b.v[j] = (float)B.v.v[j], c.v[j] = (float)C.v.v[j];
    float* const dst = &lds.bc[lane / 8][0][0].v[0] + lane % 8 * G::F;
    *reinterpret_cast<Fs<G::F>*>(dst) = b;
    *reinterpret_cast<Fs<G::F>*>(dst + G::NP) = c;
  }
};

enum Mode { kWhole, kMaps };

// What a call's states are: as many as lanes hold and decaying (with softplus), fewer, or of any number and growing.
enum Kind { kFull, kPadded, kGrowing };

// The map of a segment from its waves' maps, from the first to the last, or back: the root of its decay, and its sum.  (Decays
// meet as their logarithms: a product of what is too small with what is too large would be neither.)
template <typename G, bool BACK, typename S>
__device__ __forceinline__ void store_segment(const SelArgs& p, const S& mine, const At& at, int seg, int lane,
                                              int wave, MapLds<G>* maps, const float (&A)[G::NS], double time,
                                              const float (&sum)[G::NS]) {
  float P[G::NS], Q[G::NS];
#pragma unroll
  for (int i = 0; i < G::NS; ++i) P[i] = (float)(time * A[i]);
  maps[wave * 2].put(lane, P);
  maps[wave * 2 + 1].put(lane, sum);
  lds_barrier();
  if (wave != 0) return;
#pragma unroll
  for (int i = 0; i < G::NS; ++i) P[i] = Q[i] = 0.0f;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    const int w = BACK ? kWaves - 1 - k : k;
    float Pw[G::NS], Qw[G::NS];
    maps[w * 2].get(lane, Pw);
    maps[w * 2 + 1].get(lane, Qw);
#pragma unroll
    for (int i = 0; i < G::NS; ++i) Q[i] = apply_map<true>(run_decay<true>(Pw[i]), Qw[i], Q[i]), P[i] += Pw[i];
  }
#pragma unroll
  for (int i = 0; i < G::NS; ++i) P[i] = run_decay<true>(P[i]);
  float* const dst = p.seg + (int64_t)seg * 2 * p.batch * p.D_ * p.N;
  mine.store(p, dst, at.b, P);
  mine.store(p, dst + p.batch * p.D_ * p.N, at.b, Q);
}

// ---- forward ------------------------------------------------------------------------------------

// A workgroup carries a group of channels through a segment of time, a tile of four waves by eight steps at a time.  MAPS:
// only the segment's map is wanted; every wave then runs a quarter of the segment by itself, and their maps meet at the end.
template <typename T, typename G, Mode MODE, bool GATED, Kind KIND>
__global__ void __launch_bounds__(kWaves* kWave) selective_forward_kernel(SelArgs p) {
  constexpr int E = G::E, SL = G::SL, NS = G::NS;
  __shared__ WaveLds<G> lds_all[kWaves];
  __shared__ MapLds<G> maps[2][kWaves][2];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  WaveLds<G>& lds = lds_all[wave];
  const int seg = blockIdx.y;
  const At at = place(p, slab_of(blockIdx.x, gridDim.x), G::GROUP);
  const Slots<G, KIND != kFull> mine(p, at, lane);
  const int64_t state_size = p.batch * p.D_ * p.N;

  // the layout that memory is read and written in
  const int row = lane / 8, ec = lane % 8 * E, c = at.c0 + ec;
  const int n = G::GROUP < 8 && ec >= G::GROUP ? 0 : min(max(p.D_ - c, 0), E);
  float bias[E], skip[E], A[NS];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    bias[j] = j < n ? param<T>(p.bias, p.w32, c + j, 0.0f) : 0.0f;
    skip[j] = j < n ? param<T>(p.D, p.w32, c + j, 0.0f) : 0.0f;
  }
  mine.template rates<T>(p, A);

  const int live = (at.len + kTileSteps - 1) / kTileSteps;  // tiles that the row reaches
  const int first = seg * p.seg_tiles, last = min(first + p.seg_tiles, p.tiles), live_last = min(last, live);
  double time = 0.0;  // of the wave's steps (kMaps)
  float carry[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) carry[i] = 0.0f;
  if (MODE == kWhole) {
    if (p.h0) mine.load(p, p.h0, at.b, carry);
    for (int s = 0; s < seg; ++s) {  // the segments before this one
      float P[NS], Q[NS];
      mine.load(p, p.seg + (int64_t)s * 2 * state_size, at.b, P);
      mine.load(p, p.seg + (int64_t)(s * 2 + 1) * state_size, at.b, Q);
#pragma unroll
      for (int i = 0; i < NS; ++i) carry[i] = apply_map<true>(P[i], Q[i], carry[i]);
    }
    arrived(carry);
  }

  constexpr int kNext = MODE == kMaps ? kRun : kTileSteps;  // steps between a wave's runs
  const int start = MODE == kMaps ? (first * kWaves + wave * (last - first)) * kRun : first * kTileSteps + wave * kRun;
  const int runs = MODE == kMaps ? min(max((at.len - start + kRun - 1) / kRun, 0), last - first) : live_last - first;
  int t = start + row;  // the lane's step
  TileIn<T, G> next;
  next.place(p, at, t, c, n, lane, kNext);
  const auto load = [&](int t) __attribute__((always_inline)) {
    const bool on = t < at.len;
    next.u.load(on), next.dt.load(on), next.B.load(on);
    if (MODE == kWhole) {
      if (GATED) next.z.load(on);
      next.C.load(on);
    }
  };
  T* out = static_cast<T*>(p.out) + (at.b * p.T_ + t) * p.D_ + c;
  const int64_t out_step = (int64_t)kTileSteps * p.D_;
  if (runs > 0) load(t);
  for (int run = 0; run < runs; ++run, t += kNext, out += out_step) {
    const int tile = first + run;
    // dt and dt u, B, C: into the wave's LDS
    const Vec<T, E> u = next.u.v, z = next.z.v;
    bool odd = false;
    if (G::GROUP >= 8 || ec < G::GROUP) {
      Fs<2 * E> f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float raw = (float)next.dt.v.v[j] + bias[j], dt = t < at.len ? p.softplus ? softplus(raw) : raw : 0.0f;
        f.v[2 * j] = dt, f.v[2 * j + 1] = dt * (float)u.v[j];
        odd = odd || !__builtin_isfinite(f.v[2 * j + 1]);
      }
      *reinterpret_cast<Fs<2 * E>*>(&lds.step[row][ec]) = f;
    }
    next.put_coefs(lds, lane);
    if (run + 1 < runs) load(t + kNext);
    wave_sync();
    // 1. decays and the run's map
    float a[kRun][NS], Q[NS], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) Q[i] = MODE == kMaps ? carry[i] : 0.0f;
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
      const Fs<2> s = lds.step[r][lane / SL];
      const Fs<NS> B = lds.bc[r][0][lane % SL];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        a[r][i] = __builtin_amdgcn_exp2f(s.v[0] * A[i]);
        Q[i] = fmaf(a[r][i], Q[i], s.v[1] * B.v[i]);
      }
      sum += s.v[0];
    }
    // 2. the waves' maps
    float P[NS], h[NS] = {};
#pragma unroll
    for (int i = 0; i < NS; ++i) P[i] = run_decay<KIND == kGrowing>(sum * A[i]);
    if (MODE == kMaps) {
#pragma unroll
      for (int i = 0; i < NS; ++i) carry[i] = Q[i];
      time += sum;
      wave_sync();
      continue;
    }
    MapLds<G>(*const map)[2] = maps[tile & 1];
    map[wave][0].put(lane, P);
    map[wave][1].put(lane, Q);
    if (p.states && wave == 0) mine.store(p, p.states + tile * state_size, at.b, carry);
    lds_barrier();
    // (selects, not branches: the maps are then read one after the other without a wait)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      float Pw[NS], Qw[NS];
      map[w][0].get(lane, Pw);
      map[w][1].get(lane, Qw);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        h[i] = w == wave ? carry[i] : h[i];
        carry[i] = apply_map<KIND == kGrowing>(Pw[i], Qw[i], carry[i]);
      }
    }
    // 3. the steps from where they start
    mine.clear_missing(h), mine.clear_missing(carry);
    const auto steps = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        const Fs<2> s = lds.step[r][lane / SL];
        const Fs<NS> B = lds.bc[r][0][lane % SL], C = lds.bc[r][1][lane % SL];
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          h[i] = fmaf(a[r][i], h[i], s.v[1] * B.v[i]);
          if (decltype(careful)::value) h[i] = mine.of(i, h[i]);
          y = fmaf(C.v[i], h[i], y);
        }
        lds.y[r][lane / SL] = states_sum<SL>(y);  // (the same from all SL lanes, as below: a branch would part the steps)
      }
    };
    // (Missing states are cleared at every step only by a wave that has something infinite.  16 x 1024 x 1024 channels x 10
    // states bf16: 114 us, where every wave did it 130, without any of it 112; the backward pass, which always does, 340 and 327.)
    if (KIND != kFull && any_lane(odd))
      steps(std::bool_constant<KIND != kFull>());
    else
      steps(std::false_type());
    wave_sync();
    if (t < p.T_ && n > 0) {
      const Fs<E> sum = *reinterpret_cast<const Fs<E>*>(&lds.y[row][ec]);
      float y[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        y[j] = fmaf(skip[j], (float)u.v[j], sum.v[j]);
        if (GATED) y[j] *= silu((float)z.v[j]);
        if (t >= at.len) y[j] = 0.0f;
      }
      store_some<T, E>(out, round_to<T, E>(y), n);
    }
    wave_sync();
  }
  if (MODE == kMaps) {
    store_segment<G, false>(p, mine, at, seg, lane, wave, maps[0][0], A, time, carry);
    return;
  }
  for (int tile = max(first, live_last); tile < last; ++tile, t += kTileSteps, out += out_step)  // past the row
    if (t < p.T_) store_some<T, E>(out, Vec<T, E>{}, n);
  // (the last segment's carry is the row's: past the row nothing changes it)
  if (p.h_n && wave == 0 && seg == p.segs - 1) mine.store(p, p.h_n, at.b, carry);
}

// ---- one token ----------------------------------------------------------------------------------

// SL threads per channel with four states each.  Bound by the traffic of the states: 512 x 1024 x 16 bf16 16.8 us, 4.2
// TB/s (a copy of the states 10.1).  (Two, four and eight rows per thread, which read A once for all of them: 18.5, 18.9 and
// 31 us.)
constexpr int kStepStates = 4;
int step_lanes(int states) { return states <= 4 ? 1 : states <= 8 ? 2 : states <= 16 ? 4 : states <= 32 ? 8 : 16; }

template <typename T, int SL, bool GATED>
__global__ void __launch_bounds__(256) selective_step_kernel(SelArgs p) {
  constexpr int NS = kStepStates;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, at = i / SL;  // (less than 2^32 threads)
  const int64_t b = at / (uint32_t)p.D_;
  if (b >= p.batch) return;  // (whole groups of SL lanes)
  const int d = (int)(at % (uint32_t)p.D_), n0 = (int)(i % SL) * NS, n = min(max(p.N - n0, 0), NS);
  const int64_t state = (int64_t)at * p.N + n0;
  Vec<float, NS> h = load_some<float, NS>(p.h0 + state, n), A;
  const Vec<T, NS> B = load_some<T, NS>(static_cast<const T*>(p.B.p) + b * p.B.b + n0, n);
  const Vec<T, NS> C = load_some<T, NS>(static_cast<const T*>(p.C.p) + b * p.C.b + n0, n);
  const float u = (float)static_cast<const T*>(p.u.p)[b * p.u.b + d];
  const float raw = (float)static_cast<const T*>(p.dt.p)[b * p.dt.b + d] + param<T>(p.bias, p.w32, d, 0.0f);
  const float z = GATED ? (float)static_cast<const T*>(p.z.p)[b * p.z.b + d] : 0.0f;
  const float skip = param<T>(p.D, p.w32, d, 0.0f);
  if (p.w32) {
    A = load_some<float, NS>(static_cast<const float*>(p.A) + (int64_t)d * p.N + n0, n);
  } else {
    const Vec<T, NS> v = load_some<T, NS>(static_cast<const T*>(p.A) + (int64_t)d * p.N + n0, n);
#pragma unroll
    for (int j = 0; j < NS; ++j) A.v[j] = (float)v.v[j];
  }
  const float dt = p.softplus ? softplus(raw) : raw, du = dt * u;
  float y = 0.0f;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    h.v[j] = fmaf(__builtin_amdgcn_exp2f(dt * rate(A.v[j])), h.v[j], du * (float)B.v[j]);
    if (j < n) y = fmaf((float)C.v[j], h.v[j], y);
  }
  y = fmaf(skip, u, states_sum<SL>(y));
  if (GATED) y *= silu(z);
  store_some<float, NS>(p.h_n + state, h, n);
  if (i % SL == 0) static_cast<T*>(p.out)[at] = round_to<T>(y);
}

// ---- backward -----------------------------------------------------------------------------------

template <typename G>
struct BackLds {
  WaveLds<G> f;                          // (y: dy, then y; step: then s1, s2 of every channel)
  alignas(16) float bc[kRun][2][G::NP];  // dB and dC of the wave's channels
  // What a lane needs at both ends of a tile, of its E channels: registers that the steps in between take.
  enum Kept { kU, kDt, kDy, kRawSlope, kGateSlope, kBias, kSkip, kSumSkip, kSumBias, kKept };
  Fs<G::E> kept[kKept][64];
};

// The tiles of a segment from the last to the first.  MAPS: only the segment's map of E is wanted, as above.
template <typename T, typename G, Mode MODE, bool GATED, Kind KIND>
__global__ void __launch_bounds__(G::SIDE* kWaves* kWave, G::SIDE == 1 ? 3 : 2) selective_backward_kernel(SelArgs p) {
  constexpr int SIDE = G::SIDE, E = G::E, SL = G::SL, NS = G::NS;
  __shared__ BackLds<G> lds_all[SIDE][kWaves];
  __shared__ MapLds<G> maps[SIDE][kWaves][3];
  const int lane = threadIdx.x % kWave, id = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wave = id % kWaves, side = id / kWaves;
  BackLds<G>& back = lds_all[side][wave];
  WaveLds<G>& lds = back.f;
  const int seg = blockIdx.y;
  const int64_t slab = slab_of(blockIdx.x, gridDim.x);
  // A row's groups are taken SIDE at a time; of rows of one group each, SIDE rows.
  const bool side_rows = p.groups == 1, alone = SIDE == 1 || side_rows;  // alone: no other group's dB and dC to add
  const int per_row = (p.groups + SIDE - 1) / SIDE;
  const int64_t b_of = side_rows ? slab * SIDE + side : slab / per_row;
  const int group = side_rows ? 0 : (int)(slab % per_row) * SIDE + side;
  const bool on = b_of < p.batch && group < p.groups;
  const int sides = alone ? 1 : p.groups - (group - side);  // that have a group, where they share a row
  const At at = place(p, on ? b_of * p.groups + group : p.units, G::GROUP);
  const Slots<G, KIND != kFull> mine(p, at, lane);
  const int64_t state_size = p.batch * p.D_ * p.N;

  // B and C of the lane's states, step r's at r * kCoefs.  Those of missing channels are zeros, as their u and dy are: an
  // infinite coefficient would make them NaN, and with them dB and dC, the sums over the channels.
  constexpr int kCoefs = 2 * SL;
  __shared__ Fs<NS> none[MODE == kWhole ? kRun * kCoefs : 1];
  if (MODE == kWhole)
    for (int i = threadIdx.x; i < kRun * kCoefs; i += SIDE * kWaves * kWave) none[i] = Fs<NS>{};
  const Fs<NS>* const B_at = MODE == kMaps || mine.c < p.D_ ? &lds.bc[0][0][lane % SL] : &none[lane % SL];
  const Fs<NS>* const C_at = B_at + SL;

  const int row = lane / 8, ec = lane % 8 * E, c = at.c0 + ec;
  const int n = G::GROUP < 8 && ec >= G::GROUP ? 0 : min(max(p.D_ - c, 0), E);
  using Kept = BackLds<G>;
  const auto keep = [&](int k, const Fs<E>& v) __attribute__((always_inline)) { back.kept[k][lane] = v; };
  const auto kept = [&](int k) __attribute__((always_inline)) { return back.kept[k][lane]; };
  {
    Fs<E> bias, skip;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      bias.v[j] = j < n ? param<T>(p.bias, p.w32, c + j, 0.0f) : 0.0f;
      skip.v[j] = j < n ? param<T>(p.D, p.w32, c + j, 0.0f) : 0.0f;
    }
    keep(Kept::kBias, bias), keep(Kept::kSkip, skip), keep(Kept::kSumSkip, Fs<E>{}), keep(Kept::kSumBias, Fs<E>{});
    lds_barrier();
  }
  float A[NS];
  mine.template rates<T>(p, A);

  const auto length = [&](int64_t b) { return b >= p.batch ? 0 : p.lengths ? min(max(p.lengths[b], 0), p.T_) : p.T_; };
  const int row_len = length(b_of);  // (also of a wave without a group: it adds up its row's dB and dC)
  int most = row_len;  // the same in all waves
  if (side_rows)
    for (int i = 0; i < SIDE; ++i) most = max(most, length(slab * SIDE + i));
  const int live = (most + kTileSteps - 1) / kTileSteps;
  const int first = seg * p.seg_tiles, last = min(first + p.seg_tiles, p.tiles), live_last = min(last, live);
  double time = 0.0;
  float carry[NS], dA[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) carry[i] = dA[i] = 0.0f;
  if (MODE == kWhole) {
    if (p.d_hn) mine.load(p, p.d_hn, at.b, carry);
    for (int s = p.segs - 1; s > seg; --s) {  // the segments after this one
      float P[NS], Q[NS];
      mine.load(p, p.seg + (int64_t)s * 2 * state_size, at.b, P);
      mine.load(p, p.seg + (int64_t)(s * 2 + 1) * state_size, at.b, Q);
#pragma unroll
      for (int i = 0; i < NS; ++i) carry[i] = apply_map<true>(P[i], Q[i], carry[i]);
    }
    arrived(carry);
  }

  constexpr int kNext = MODE == kMaps ? kRun : kTileSteps;  // steps between a wave's runs
  const int start = MODE == kMaps ? (first * kWaves + wave * (last - first)) * kRun : first * kTileSteps + wave * kRun;
  const int runs = MODE == kMaps ? min(max((at.len - start + kRun - 1) / kRun, 0), last - first) : live_last - first;
  int t = start + (runs - 1) * kNext + row;  // the lane's step
  TileIn<T, G> next;
  Rows<T, E> next_g;
  next.place(p, at, t, c, n, lane, -kNext);
  next_g.place(Strided{p.d_out, (int64_t)p.T_ * p.D_, p.D_}, at.b, t, c, n, -kNext);
  const auto load = [&](int t) __attribute__((always_inline)) {
    const bool on = t < at.len;
    next_g.load(on), next.dt.load(on), next.C.load(on);
    if (GATED) next.z.load(on);
    if (MODE == kWhole) next.u.load(on), next.B.load(on);
  };
  // dB and dC of a tile that is done (its waves have met at a barrier since)
  const int64_t bc_group = side_rows ? 0 : slab % per_row;
  const int f = lane % 8 * G::F, f_states = G::NP < 8 && f >= G::NP ? 0 : min(max(p.N - f, 0), G::F);
  const auto flush = [&](int t) __attribute__((always_inline)) {
    if (t >= row_len) return;
    float* const dst = p.part_bc + ((bc_group * p.batch + b_of) * p.T_ + t) * 2 * p.N + f;
    const auto of = [&](int side, int k) __attribute__((always_inline)) {
      return *reinterpret_cast<const Fs<G::F>*>(&lds_all[side][wave].bc[row][k][f < G::NP ? f : 0]);
    };
    const auto put = [&](int k, const Fs<G::F>& v) __attribute__((always_inline)) {
      store_some<float, G::F>(dst + k * p.N, __builtin_bit_cast(FVec<G::F>, v), f_states);
    };
    if (alone) {
      put(0, of(side, 0)), put(1, of(side, 1));
    } else if (side < 2) {  // a row's sums: dB by the first side's waves, dC by the second one's
      Fs<G::F> v = of(0, side);
#pragma unroll
      for (int i = 1; i < SIDE; ++i) {
        if (i >= sides) break;
        const Fs<G::F> other = of(i, side);
#pragma unroll
        for (int j = 0; j < G::F; ++j) v.v[j] += other.v[j];
      }
      put(side, v);
    }
  };
  if (runs > 0) load(t);
  for (int run = runs - 1; run >= 0; --run, t -= kNext) {
    const int tile = first + run;
    float h[NS];
    if (MODE == kWhole) {
#pragma unroll
      for (int i = 0; i < NS; ++i) h[i] = 0.0f;
      if (tile * kTileSteps < at.len) mine.load(p, p.states + tile * state_size, at.b, h);
    }
    {
      const bool in = t < at.len;
      const Fs<E> bias = kept(Kept::kBias);
      Fs<E> u, dt, dy, d_raw, d_gate;  // (d_raw: the slope of dt; d_gate: the output's by z, but for the factor y)
      Fs<2 * E> f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        u.v[j] = (float)next.u.v.v[j];
        dt.v[j] = (float)next.dt.v.v[j] + bias.v[j], d_raw.v[j] = 1.0f;
        if (p.softplus) softplus(dt.v[j], dt.v[j], d_raw.v[j]);
        if (!in) dt.v[j] = 0.0f;
        dy.v[j] = (float)next_g.v.v[j];
        if (GATED) {
          float value, slope;
          silu((float)next.z.v.v[j], value, slope);
          d_gate.v[j] = dy.v[j] * slope, dy.v[j] *= value;
        }
        f.v[2 * j] = dt.v[j], f.v[2 * j + 1] = dt.v[j] * u.v[j];
      }
      if (MODE == kWhole) {
        keep(Kept::kU, u), keep(Kept::kDt, dt), keep(Kept::kDy, dy), keep(Kept::kRawSlope, d_raw);
        if (GATED) keep(Kept::kGateSlope, d_gate);
      }
      if (G::GROUP >= 8 || ec < G::GROUP) {
        *reinterpret_cast<Fs<2 * E>*>(&lds.step[row][ec]) = f;
        *reinterpret_cast<Fs<E>*>(&lds.y[row][ec]) = dy;
      }
    }
    next.put_coefs(lds, lane);
    if (run > 0) load(t - kNext);
    wave_sync();
    // 1. decays, the run's maps forward (h) and backward (E)
    float a[kRun][NS], Qh[NS], Qe[NS], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) Qh[i] = 0.0f, Qe[i] = MODE == kMaps ? carry[i] : 0.0f;
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
      const Fs<2> s = lds.step[r][lane / SL];
      const Fs<NS> B = B_at[r * kCoefs];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        a[r][i] = __builtin_amdgcn_exp2f(s.v[0] * A[i]);
        if (MODE == kWhole) Qh[i] = fmaf(a[r][i], Qh[i], s.v[1] * B.v[i]);
      }
      sum += s.v[0];
    }
#pragma unroll
    for (int r = kRun - 1; r >= 0; --r) {
      const Fs<NS> C = C_at[r * kCoefs];
      const float q = lds.y[r][lane / SL];
#pragma unroll
      for (int i = 0; i < NS; ++i) Qe[i] = a[r][i] * fmaf(C.v[i], q, Qe[i]);
    }
    // 2. the waves' maps
    float P[NS], e[NS] = {};
#pragma unroll
    for (int i = 0; i < NS; ++i) P[i] = run_decay<KIND == kGrowing>(sum * A[i]);
    if (MODE == kMaps) {
#pragma unroll
      for (int i = 0; i < NS; ++i) carry[i] = Qe[i];
      time += sum;
      wave_sync();
      continue;
    }
    MapLds<G>(*const map)[3] = maps[side];
    map[wave][0].put(lane, P);
    map[wave][1].put(lane, Qe);
    map[wave][2].put(lane, Qh);
    lds_barrier();
    if (run + 1 < runs) flush(t + kTileSteps);
    // (selects, not branches: the maps are then read one after the other without a wait)
#pragma unroll
    for (int w = kWaves - 1; w >= 0; --w) {
      float Pw[NS], Qw[NS];
      map[w][0].get(lane, Pw);
      map[w][1].get(lane, Qw);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        e[i] = w == wave ? carry[i] : e[i];
        carry[i] = apply_map<KIND == kGrowing>(Pw[i], Qw[i], carry[i]);
      }
    }
#pragma unroll
    for (int w = 0; w + 1 < kWaves; ++w) {
      float Pw[NS], Qw[NS];
      map[w][0].get(lane, Pw);
      map[w][2].get(lane, Qw);
#pragma unroll
      for (int i = 0; i < NS; ++i) h[i] = w < wave ? apply_map<KIND == kGrowing>(Pw[i], Qw[i], h[i]) : h[i];
    }
    lds_barrier();  // (the maps and the sums of the tile before have been read)
    mine.clear_missing(h), mine.clear_missing(e), mine.clear_missing(carry);
    // 3. the states, each before its step
    float before[kRun + 1][NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) before[0][i] = h[i];
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
      const Fs<2> s = lds.step[r][lane / SL];
      const Fs<NS> B = B_at[r * kCoefs];
#pragma unroll
      for (int i = 0; i < NS; ++i)
        before[r + 1][i] = mine.of(i, fmaf(a[r][i], before[r][i], s.v[1] * B.v[i]));
    }
    wave_sync();  // (or what the steps read would be kept in registers for the way back)
    // 4. and backwards through them
    const auto walk = [&](auto whole) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
      for (int r = kRun - 1; r >= 0; --r) {
        // (past the row E stays as it is, and a product of what is infinite there with a zero must not count)
        if (!WHOLE && tile * kTileSteps + wave * kRun + r >= at.len) continue;
        const Fs<2> s = lds.step[r][lane / SL];
        const Fs<NS> B = B_at[r * kCoefs], C = C_at[r * kCoefs];
        const float q = lds.y[r][lane / SL];
        float s1 = 0.0f, s2 = 0.0f, y = 0.0f, dB[NS], dC[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const float g = mine.of(j, fmaf(C.v[j], q, e[j]));
          s1 = fmaf(g, B.v[j], s1);
          dB[j] = g * s.v[1];
          dC[j] = q * before[r + 1][j];
          if (GATED) y = fmaf(C.v[j], before[r + 1][j], y);
          e[j] = a[r][j] * g;
          const float m = e[j] * before[r][j];
          s2 = fmaf(m, A[j], s2);
          dA[j] = fmaf(m, s.v[0], dA[j]);
        }
        lds.step[r][lane / SL] = Fs<2>{{states_sum<SL>(s1), states_sum<SL>(s2)}};
        if (GATED) lds.y[r][lane / SL] = states_sum<SL>(y);
        // dB to the low half of the wave, dC to the high one; with four states 0, 2 to the even rows of 16 lanes and 1, 3 to
        // the odd ones, with two 0 and 1
        float w[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) w[j] = pair_sum<true>(dB[j], dC[j]);
        float* const dst = &back.bc[r][lane / 32][lane % SL * NS + (NS > 1 ? lane / 16 % 2 : 0)];
        if constexpr (NS == 4) {
          const float x0 = row_rest_sum<SL>(pair_sum<false>(w[0], w[1])), x2 = row_rest_sum<SL>(pair_sum<false>(w[2], w[3]));
          // (from all lanes: a condition on the lane, which is a branch, costs 1330 us where this takes 605)
          if constexpr (SL <= 8)
            dst[lane & 8 ? 2 : 0] = lane & 8 ? x2 : x0;
          else
            dst[0] = x0, dst[2] = x2;
        } else {
          const float x0 = row_rest_sum<SL>(pair_sum<false>(w[0], w[NS - 1]));
          dst[0] = x0;
        }
      }
    };
    if (tile * kTileSteps + (wave + 1) * kRun <= at.len)
      walk(std::true_type());
    else
      walk(std::false_type());
    wave_sync();
    if (t < p.T_ && n > 0) {
      const bool in = t < at.len;
      const Fs<2 * E> f = *reinterpret_cast<const Fs<2 * E>*>(&lds.step[row][ec]);
      const Fs<E> y = *reinterpret_cast<const Fs<E>*>(&lds.y[row][ec]), skip = kept(Kept::kSkip);
      const Fs<E> u = kept(Kept::kU), dt = kept(Kept::kDt), dy = kept(Kept::kDy), d_raw = kept(Kept::kRawSlope);
      Fs<E> d_gate = {}, d_skip = kept(Kept::kSumSkip), d_bias = kept(Kept::kSumBias);
      if (GATED) d_gate = kept(Kept::kGateSlope);
      float du[E], dr[E], dz[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        constexpr float kLn2 = 0.69314718f;
        du[j] = in ? fmaf(dt.v[j], f.v[2 * j], dy.v[j] * skip.v[j]) : 0.0f;
        dr[j] = in ? fmaf(u.v[j], f.v[2 * j], f.v[2 * j + 1] * kLn2) * d_raw.v[j] : 0.0f;
        dz[j] = in ? d_gate.v[j] * fmaf(skip.v[j], u.v[j], y.v[j]) : 0.0f;
        if (in) d_skip.v[j] = fmaf(dy.v[j], u.v[j], d_skip.v[j]);
        d_bias.v[j] += dr[j];
      }
      keep(Kept::kSumSkip, d_skip), keep(Kept::kSumBias, d_bias);
      const int64_t o = (at.b * p.T_ + t) * p.D_ + c;
      store_some<T, E>(static_cast<T*>(p.d_u) + o, round_to<T, E>(du), n);
      store_some<T, E>(static_cast<T*>(p.d_dt) + o, round_to<T, E>(dr), n);
      if (GATED) store_some<T, E>(static_cast<T*>(p.d_z) + o, round_to<T, E>(dz), n);
    }
    wave_sync();
  }
  if (MODE == kMaps) {
    store_segment<G, true>(p, mine, at, seg, lane, wave, maps[side][0], A, time, carry);
    return;
  }
  for (int tile = max(first, live_last); tile < last; ++tile) {  // past the row
    const int t = tile * kTileSteps + wave * kRun + row;
    if (t >= p.T_ || n <= 0) continue;
    const int64_t o = (at.b * p.T_ + t) * p.D_ + c;
    store_some<T, E>(static_cast<T*>(p.d_u) + o, Vec<T, E>{}, n);
    store_some<T, E>(static_cast<T*>(p.d_dt) + o, Vec<T, E>{}, n);
    if (GATED) store_some<T, E>(static_cast<T*>(p.d_z) + o, Vec<T, E>{}, n);
  }
  if (p.d_h0 && wave == 0 && seg == 0) mine.store(p, p.d_h0, at.b, carry);

  // The waves' sums of dA, dD and dbias, added in their order.
  lds_barrier();
  if (first < live_last) flush(first * kTileSteps + wave * kRun + row);
  lds_barrier();
  float* const part = p.part_w + ((int64_t)seg * p.batch + at.b) * p.D_ * (p.N + 2);
  maps[side][wave][0].put(lane, dA);
  lds_barrier();
  if (wave == 0) {
    float v[NS];
    for (int w = 1; w < kWaves; ++w) {
      maps[side][w][0].get(lane, v);
#pragma unroll
      for (int i = 0; i < NS; ++i) dA[i] += v[i];
    }
    mine.store(p, part - at.b * p.D_ * p.N, at.b, dA);
  } else if (wave == 1 && lane < 16) {
    // eight lanes with E channels each, for dD and for dbias, over the lanes that share a channel: the eight rows
    const int k = lane / 8;
    Vec<float, E> v = {};
    for (int w = 0; w < kWaves; ++w) {
      for (int r = 0; r < 8; ++r) {
        const Fs<E> t = lds_all[side][w].kept[Kept::kSumSkip + k][r * 8 + lane % 8];
#pragma unroll
        for (int j = 0; j < E; ++j) v.v[j] += t.v[j];
      }
    }
    store_some<float, E>(part + (int64_t)p.D_ * (p.N + k) + c, v, n);
  }
}

// dB and dC: the workgroups' sums, in their order (of four neighbouring ones per thread: 57.5 us against 61.5 at
// 8 x 2048 x 2048 x 16 states, 27.3 against 26.8 at 128 x 1000 x 256 ragged: left as it is).
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

// f(std::integral_constant of the lanes, and of the states per lane) that serve `states`.
template <typename F>
auto with_states(int states, F&& f) {
  if (states <= 4) return f(std::integral_constant<int, 4>(), std::integral_constant<int, 1>());
  if (states <= 8) return f(std::integral_constant<int, 4>(), std::integral_constant<int, 2>());
  if (states <= 16) return f(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
  if (states <= 32) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 4>());
  return f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
}

struct SelLayout {
  int groups;     // of channels, in a row
  int tiles, seg_tiles, segs;
  int bc_groups;  // sums of dB and dC
};

// With few workgroups the time axis is split into segments, whose maps a launch of its own computes first (about half of
// the work again).  Workgroups that fill the device, at as many registers as they take: 1024 forward, 768 backward (256 with
// two groups each).  Measured, us of a call without and with about that many, 16 states bf16 with a gate:
//   forward   64 workgroups (2 x 4096 x 512) 264 and 58, 80 (1 x 16384 x 1280) 1177 and 284, 128 (1 x 2048 x 2048)
//             134 and 58, 256 (4 x 2048 x 1024) 153 and 99; 512 (4 x 2048 x 2048) 162, in two segments 174
//   backward  64 594 and 122, 80 2483 and 616, 128 316 and 132, 256 312 and 209; 512 427, in two segments 487
SelLayout sel_layout(int64_t batch, int64_t seq_len, int64_t channels, int states, bool backward) {
  SelLayout l;
  int per = 0, side = 0;
  with_states(states, [&](auto sl, auto ns) {
    using G = Geo<decltype(sl)::value, decltype(ns)::value>;
    per = G::GROUP, side = G::SIDE;
  });
  l.groups = (int)((channels + per - 1) / per);
  l.bc_groups = (l.groups + side - 1) / side;
  l.tiles = (int)((seq_len + kTileSteps - 1) / kTileSteps);
  const int64_t units = batch * l.groups, slabs = l.groups == 1 ? (batch + side - 1) / side : batch * l.bc_groups;
  const int64_t groups = std::max<int64_t>(1, backward ? slabs : units);  // of workgroups
  const int64_t fill = backward ? side == 1 ? 768 : 256 : 1024, most = backward ? fill / 2 : 400;
  const int64_t want = groups > most ? 1 : fill / groups;
  // (no segment shorter than two tiles: a short one's start costs as much as its steps)
  l.seg_tiles = (int)std::max<int64_t>(std::max(1, std::min(2, l.tiles)), (l.tiles + want - 1) / want);
  l.segs = std::max(1, (l.tiles + l.seg_tiles - 1) / l.seg_tiles);
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

// f(std::integral_constant of the kind of states), of which lanes hold `padded`.
template <typename F>
hipError_t with_kind(const SelArgs& p, int padded, F&& f) {
  if (!p.softplus) return f(std::integral_constant<Kind, kGrowing>());
  return p.N < padded ? f(std::integral_constant<Kind, kPadded>()) : f(std::integral_constant<Kind, kFull>());
}

template <typename T>
hipError_t launch_sel_forward(const SelArgs& p, hipStream_t s) {
  return with_states(p.N, [&](auto sl, auto ns) {
    using G = Geo<decltype(sl)::value, decltype(ns)::value>;
    const dim3 block(kWaves * kWave);
    if (p.segs > 1) {
      const dim3 all_but_last((unsigned)p.units, p.segs - 1);
      hipLaunchKernelGGL((selective_forward_kernel<T, G, kMaps, false, kFull>), all_but_last, block, 0, s, p);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return with_kind(p, G::NP, [&](auto kind) {
      constexpr Kind KIND = decltype(kind)::value;
      const dim3 grid((unsigned)p.units, p.segs);
      if (p.z.p)
        hipLaunchKernelGGL((selective_forward_kernel<T, G, kWhole, true, KIND>), grid, block, 0, s, p);
      else
        hipLaunchKernelGGL((selective_forward_kernel<T, G, kWhole, false, KIND>), grid, block, 0, s, p);
      return hipGetLastError();
    });
  });
}

template <typename T>
hipError_t launch_sel_step(const SelArgs& p, hipStream_t s) {
  const auto run = [&](auto lanes) {
    constexpr int SL = decltype(lanes)::value;
    const dim3 grid((unsigned)((p.batch * p.D_ * SL + 255) / 256));
    if (p.z.p)
      hipLaunchKernelGGL((selective_step_kernel<T, SL, true>), grid, dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((selective_step_kernel<T, SL, false>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
  };
  switch (step_lanes(p.N)) {
    case 1: return run(std::integral_constant<int, 1>());
    case 2: return run(std::integral_constant<int, 2>());
    case 4: return run(std::integral_constant<int, 4>());
    case 8: return run(std::integral_constant<int, 8>());
    default: return run(std::integral_constant<int, 16>());
  }
}

template <typename T>
hipError_t launch_sel_backward(SelArgs p, void* d_A, void* d_B, void* d_C, void* d_D, void* d_bias, hipStream_t s) {
  hipError_t e = hipSuccess;
  if (p.batch > 0) {
    e = with_states(p.N, [&](auto sl, auto ns) {
      using G = Geo<decltype(sl)::value, decltype(ns)::value>;
      const int64_t slabs = p.groups == 1 ? (p.batch + G::SIDE - 1) / G::SIDE : p.batch * p.bc_groups;
      const dim3 grid((unsigned)slabs, p.segs), block(G::SIDE * kWaves * kWave);
      const auto run = [&](auto gated) {
        constexpr bool GATED = decltype(gated)::value;
        if (p.segs > 1) {
          hipLaunchKernelGGL((selective_backward_kernel<T, G, kMaps, GATED, kFull>), grid, block, 0, s, p);
          const hipError_t e2 = hipGetLastError();
          if (e2 != hipSuccess) return e2;
        }
        return with_kind(p, G::NP, [&](auto kind) {
          hipLaunchKernelGGL((selective_backward_kernel<T, G, kWhole, GATED, decltype(kind)::value>), grid, block, 0, s, p);
          return hipGetLastError();
        });
      };
      return p.z.p ? run(std::true_type()) : run(std::false_type());
    });
    const int64_t n = p.batch * p.T_ * 2 * p.N;
    if (e == hipSuccess && n > 0 && (d_B || d_C)) {
      const dim3 grid((unsigned)((n + 255) / 256));
      hipLaunchKernelGGL(selective_coefs_kernel<T>, grid, dim3(256), 0, s, p, (T*)d_B, (T*)d_C);
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

int check_selective(const char* what, const plh_selective_scan_args* a, bool step) noexcept {
  if (!a) return op_error(PLH_ERR_INVALID, what, "args is required");
  if (a->dtype != PLH_F16 && a->dtype != PLH_BF16 && a->dtype != PLH_F32)
    return op_error(PLH_ERR_INVALID, what, "dtype must be PLH_F16, PLH_BF16 or PLH_F32");
  if (a->wdtype != a->dtype && a->wdtype != PLH_F32)
    return op_error(PLH_ERR_INVALID, what, "wdtype must be dtype or PLH_F32");
  if (a->batch < 0 || a->seq_len < 0) return op_error(PLH_ERR_INVALID, what, "batch and seq_len must be non-negative");
  if (a->states < 1 || a->states > kMaxStates) return op_error(PLH_ERR_UNSUPPORTED, what, "states must lie in [1, 64]");
  if (a->channels < 1 || a->channels > (1 << 20))
    return op_error(PLH_ERR_UNSUPPORTED, what, "channels must lie in [1, 2^20]");
  if (a->seq_len > (1 << 30)) return op_error(PLH_ERR_UNSUPPORTED, what, "seq_len must not exceed 2^30");
  // (a launch has fewer than 2^32 threads, in whole workgroups of 256)
  if (step && (a->batch > (int64_t(1) << 32) || a->batch * a->channels * step_lanes(a->states) > (int64_t(1) << 32) - 256))
    return op_error(PLH_ERR_UNSUPPORTED, what, "batch * channels * lanes per channel must not exceed 2^32 - 256");
  // (Both directions' launches stay below 2^32 threads: a workgroup of 256 has 16 channels with up to 16 states, then 8, then
  // 4; one of 512, the backward pass's with more than 16 states, twice as many.  What remains beside the second limit, 2^21
  // rows and more of up to eight channels, has 2^30.)
  const int64_t eights = a->batch > (1 << 23) ? int64_t(1) << 23 : a->batch * ((a->channels + 7) / 8);
  if (!step && eights > (a->batch < (1 << 21) ? (1 << 23) - 1 : 1 << 21))
    return op_error(PLH_ERR_UNSUPPORTED, what,
                    "batch * ceil(channels / 8) must be below 2^23, and from 2^21 rows on not exceed 2^21");
  if (!step && a->batch * a->seq_len * a->states > (1 << 30))
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
  if (batch < 0 || seq_len < 0 || seq_len > (1 << 30) || channels < 1 || channels > (1 << 20) || states < 1 ||
      states > plh::kMaxStates)
    return -1;
  return plh::sel_workspace(batch, seq_len, channels, states, backward != 0).bytes;
}

int plh_selective_scan_forward(const plh_selective_scan_args* a, const float* h0, void* out, float* h_n, float* states,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* const what = "selective_scan_forward";
  const int rc = plh::check_selective(what, a, false);
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
  const int rc = plh::check_selective(what, a, true);
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
  const int rc = plh::check_selective(what, a, false);
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
