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

// A workgroup carries a slab of channels through time, a tile of steps at a time.  A thread has VEC neighbouring channels
// for R consecutive steps; CT threads side by side read one step of the slab, the TG groups of so many threads are
// consecutive in time.  A row's channels are cut into pieces of VEC, the last of which is moved back to end with the
// row: its channels are then carried by two threads, which compute and store the same.  Pieces are numbered row after
// row, so that slabs are full whatever H is.
constexpr int kTile = 64;  // steps of a tile where there can be several (MANY): its loads are then in flight one ahead
template <int VEC, int CT, int TG, int R, bool MANY>
struct Place;
using Usual = Place<4, 16, 16, 4, true>;     // 256 threads, 64 channels, 64 steps
using Wide = Place<4, 32, 16, 4, true>;      // 512 threads, 128 channels, 64 steps (see layout_for)
using Narrow = Place<1, 64, 4, 16, true>;    // 256 threads, 64 channels, 64 steps: H < 4
using Steps64 = Place<4, 16, 16, 4, false>;  // 256 threads and one tile: 64 channels, 64 steps,
using Steps32 = Place<4, 32, 8, 4, false>;   // 128 channels, 32 steps,
using Steps16 = Place<4, 64, 4, 4, false>;   // 256 channels, 16 steps

template <typename T>
struct ScanArgs {
  const T* gates;
  int64_t stride_b, stride_t;  // elements
  int64_t channels;            // B H
  int T_, H, tiles, seg_tiles, segs;
  unsigned slabs, pieces;
  int ct;
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

// The slab of a launch's workgroup i of n.  Workgroups go round the eight XCDs in turn; here each XCD gets neighbouring
// slabs, so that a cache line that two slabs share is read into one L2 (33 x 1001 x 333 fp16, no slab aligned: forward
// 47.7 -> 40.2 us, backward 79.4 -> 68.2).
__device__ __forceinline__ unsigned slab_of(unsigned i, unsigned n) {
  const unsigned per = n / 8;
  return i < per * 8 ? (i % 8) * per + i / 8 : i;
}

// Where a thread stands: its channels, its place among the time groups, its row's length.
template <int VEC_, int CT_, int TG_, int R_, bool MANY_>
struct Place {
  static constexpr int VEC = VEC_, CT = CT_, TG = TG_, R = R_;
  static constexpr bool MANY = MANY_;
  static constexpr int TILE = TG * R, THREADS = CT * TG, WAVES = THREADS / kWave, SLAB = CT * VEC;
  static_assert(CT == 16 || CT == 32 || CT == 64, "four, two or one time groups in a wave");
  static_assert(TILE == kTile || (!MANY && TILE < kTile), "states are stored every kTile steps");
  int lane, wave, ct, tg;
  bool on;
  int64_t b, n;  // row; first channel, counted over all rows
  int h, len;
  int live_tiles;  // tiles that a row of the slab reaches (the same in every wave: each has all of the slab's channels)

  template <typename T>
  __device__ __forceinline__ Place(const ScanArgs<T>& p, unsigned slab) {
    const int tid = threadIdx.x;
    lane = tid % kWave, ct = tid % CT, tg = tid / CT;
    wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t per = (p.H + VEC - 1) / VEC, piece = slab * CT + ct;  // (batch * hidden <= 2^29)
    on = piece < p.pieces;
    b = 0, n = 0, h = 0, len = 0;
    if (on) {
      b = piece / per;
      h = min((int)(piece % per) * VEC, p.H - VEC);
      n = b * p.H + h;
      len = p.T_;
      if (p.lengths) len = min(max(p.lengths[b], 0), p.T_);
    }
    int most = len;
#pragma unroll
    for (int d = 1; d < CT; d *= 2) most = max(most, __shfl_xor(most, d));
    live_tiles = __builtin_amdgcn_readfirstlane((most + TILE - 1) / TILE);
  }
};

// Channels per thread.
inline int scan_vec(int64_t hidden) { return hidden >= 4 ? 4 : 1; }

int64_t pieces_of(int64_t batch, int64_t hidden) { return batch * ((hidden + scan_vec(hidden) - 1) / scan_vec(hidden)); }

// How a call is laid out on the device.
struct Layout {
  int ct;         // the slabs' CT
  int64_t slabs;
  int tiles;      // tiles of a row
  int seg_tiles;  // ... of a segment
  int segs;       // segments of the time axis
};

// Up to 64 steps take one tile of a size that they fill (forward / backward us; where every call has tiles of 64 steps and
// room for the next one's loads, and here): 300 rows of 512 bf16, 16 steps 15.7 / 24.5 and 7.3 / 11.1, 32 steps
// 16.5 / 27.9 and 10.2 / 17.6, 33 steps 16.9 / 28.1 and 14.8 / 23.2, 64 steps 19.6 / 36.2 and 18.3 / 35.8; 400 x 15 x 400
// fp32 17.0 / 36.0 and 7.8 / 12.2.
// More steps: with few slabs the time axis is split into segments, whose maps a launch of its own computes first.  Rows of 16-bit
// elements may be read 256 bytes at a time, in wide slabs, instead of 128 (as 32-bit ones are in the usual slabs).
// Measured, us, on 256 CUs, by the number of usual slabs (forward / backward; bf16 or fp16 with output gate):
//   352 and more: no split; wide slabs, but not where the last round of their workgroups, one per CU, would be far from
//     full.  usual -> wide: 512 slabs 235 / 411 -> 216 / 353 (16 x 4096 x 2048), B x 1000 x 256 with 360 slabs
//     58 / 84 -> 53 / 76, 512 61 / 101 -> 59 / 99, 600 76 / 138 -> 85 / 153, 800 107 / 172 -> 97 / 158, 1200
//     151 / 230 -> 152 / 244, 2000 233 / 371 -> 219 / 359;  rows that no line divides, 300 x 2493 x 88 (413):
//     158 / 348 -> 145 / 277, in two segments 207 / 401
//   160 to 351: usual slabs; forward about 768 workgroups (300 slabs with 1, 2, 3, 4 segments: 111, 99, 90, 95),
//     backward no split (256: 109, 125, 143, 143; 192: 104, 110, 111, 115)
//   32 to 159: wide slabs for 16 bits; forward 512 workgroups, backward 256.  usual -> wide: 64 slabs 46 / 76 ->
//     40 / 72, 128 62 / 108 -> 57 / 93, 61 (4 x 12837 x 968) 152 / 289 -> 150 / 254
//   fewer: usual slabs, 768 and 512 workgroups.  20 slabs (2 x 16384 x 640) with 256, 512, 768 workgroups: 85 / 117,
//     57 / 100, 53 / 95; in wide slabs 54 / 109
Layout layout_for(int elem_bytes, int64_t batch, int64_t seq_len, int64_t hidden, bool backward) {
  const int64_t pieces = std::max<int64_t>(pieces_of(batch, hidden), 1);
  if (hidden >= 4 && seq_len <= kTile) {
    const int ct = seq_len <= Steps16::TILE ? Steps16::CT : seq_len <= Steps32::TILE ? Steps32::CT : Steps64::CT;
    return {ct, (pieces + ct - 1) / ct, seq_len > 0, 1, 1};
  }
  Layout l;
  l.ct = hidden >= 4 ? Usual::CT : Narrow::CT;
  const int64_t usual = (pieces + l.ct - 1) / l.ct, wide = (pieces + 31) / 32, rounds = (wide + 255) / 256;
  const bool may = elem_bytes == 2 && hidden >= 4;
  int groups = 0;  // (no split)
  bool take_wide = false;
  if (usual >= 352) {
    take_wide = may && (rounds == 1 || 4 * wide >= 3 * 256 * rounds);
  } else if (usual >= 160) {
    if (!backward) groups = 768;
  } else if (usual >= 32 && may) {
    take_wide = true;
    groups = backward ? 256 : 512;
  } else {
    groups = backward ? 512 : 768;
  }
  if (take_wide) l.ct = Wide::CT;
  l.slabs = take_wide ? wide : usual;
  l.tiles = (int)((seq_len + kTile - 1) / kTile);
  const int want = std::max(1, (int)((groups + l.slabs / 2) / l.slabs));
  l.seg_tiles = std::max(1, (l.tiles + want - 1) / want);
  l.segs = std::max(1, (l.tiles + l.seg_tiles - 1) / l.seg_tiles);
  return l;
}

// A factor of a map that is composed of several steps.  Every step's own is positive (at least 2^-126, see logistic()), so
// that an infinite state stays infinite; their product may underflow, and 0 * inf would be NaN.  Held at 2^-126 it moves
// a finite state by less than 2^-126 of what it was.  (A NaN factor is dropped here: the map's sum holds it as well.)
__device__ __forceinline__ float factor(float a) { return __builtin_fmaxf(a, 0x1p-126f); }
template <int VEC>
__device__ __forceinline__ void hold_factors(float (&A)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) A[j] = factor(A[j]);
}

// v of the even and of the odd time group of a pair of groups, in both (one exchange per level and value).
template <int LEVEL>
__device__ __forceinline__ void pair_of(float v, float& even, float& odd) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  uint32_t lo, hi;
  if constexpr (LEVEL == 0) {  // groups of 16 lanes: neighbouring rows
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
template <typename P, int SUMS, bool REVERSE0, int VEC = P::VEC>
__device__ __forceinline__ void wave_maps(int lane, float (&A)[VEC], float (&B)[SUMS][VEC], float (&pa)[SUMS][VEC],
                                          float (&pb)[SUMS][VEC]) {
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) pa[k][j] = 1.0f, pb[k][j] = 0.0f;
  const auto level = [&](auto lv) {
    constexpr int L = decltype(lv)::value;
    const bool odd = (lane & (L == 0 ? 16 : 32)) != 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float a0, a1;
      pair_of<L>(A[j], a0, a1);
#pragma unroll
      for (int k = 0; k < SUMS; ++k) {
        const bool rev = REVERSE0 || k == 1;
        float b0, b1;
        pair_of<L>(B[k][j], b0, b1);
        // the other group of the pair comes first for the odd one in order, for the even one in reverse
        const float fa = rev ? a1 : a0, fb = rev ? b1 : b0, sa = rev ? a0 : a1, sb = rev ? b0 : b1;
        if (odd != rev) {
          pb[k][j] = fmaf(pa[k][j], fb, pb[k][j]);
          pa[k][j] = factor(pa[k][j] * fa);
        }
        B[k][j] = fmaf(sa, fb, sb);
      }
      A[j] = factor(a0 * a1);
    }
  };
  if constexpr (P::CT == 16) level(std::integral_constant<int, 0>());
  if constexpr (P::CT <= 32) level(std::integral_constant<int, 1>());
}

// The waves' maps in LDS: [parity of the tile][wave][A, sums...][channel].  Two halves in turn need one barrier
// per tile: the half written next was last read before the barrier in between.
struct alignas(16) Lds4 {
  float v[4];
};
template <int VEC>
__device__ __forceinline__ void put_lds(float* dst, const float (&v)[VEC]) {
  if constexpr (VEC == 4)
    *reinterpret_cast<Lds4*>(dst) = Lds4{{v[0], v[1], v[2], v[3]}};
  else
    dst[0] = v[0];
}
template <int VEC>
__device__ __forceinline__ Vec<float, VEC> get_lds(const float* src) {
  if constexpr (VEC == 4) {
    const Lds4 r = *reinterpret_cast<const Lds4*>(src);
    return {{r.v[0], r.v[1], r.v[2], r.v[3]}};
  } else {
    return {{src[0]}};
  }
}
template <typename P, int SUMS>
using TileMaps = float[P::WAVES][1 + SUMS][P::SLAB];
template <typename P, int SUMS>
using WaveMaps = TileMaps<P, SUMS>[2];

template <typename P, int SUMS, int VEC = P::VEC>
__device__ __forceinline__ void put_maps(const P& at, TileMaps<P, SUMS>& lds, const float (&A)[VEC],
                                         const float (&B)[SUMS][VEC]) {
  if (at.lane < P::CT) {
    put_lds<VEC>(&lds[at.wave][0][at.ct * VEC], A);
#pragma unroll
    for (int k = 0; k < SUMS; ++k) put_lds<VEC>(&lds[at.wave][1 + k][at.ct * VEC], B[k]);
  }
}

// The carry through the waves' maps: `carry` becomes the value after the whole tile, `mine` the value that this
// thread's steps start from; (pa, pb) is the thread's map from wave_maps.
template <typename P, int SUMS, int K, bool REVERSE, int VEC = P::VEC>
__device__ __forceinline__ void fold_waves(const P& at, const TileMaps<P, SUMS>& lds, const float (&pa)[VEC],
                                           const float (&pb)[VEC], float (&carry)[VEC], float (&mine)[VEC]) {
  constexpr int W = P::WAVES;
  float before[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) before[j] = carry[j];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int w = REVERSE ? W - 1 - i : i;
    if (i > 0 && w == at.wave) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) before[j] = carry[j];
    }
    const Vec<float, VEC> a = get_lds<VEC>(&lds[w][0][at.ct * VEC]), b = get_lds<VEC>(&lds[w][1 + K][at.ct * VEC]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) carry[j] = fmaf(a.v[j], carry[j], b.v[j]);
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) mine[j] = fmaf(pa[j], before[j], pb[j]);
}

// Forward, the carry goes from wave to wave, and from the last one to the first one's next tile: slot[w] holds what
// wave w starts its part of a tile from, tag[w] the number of the tile (from 1 on, in the order of the scan) that it is
// for.  A wave waits for the one before it alone, so that the waves of a workgroup do not run in step as they would
// around a barrier: half of them load and store while the others compute (16 x 4096 x 2048 bf16 forward 243 -> 235 us,
// and with 128-channel slabs, which lose without it, 215).  (The backward pass, where c and E go through a tile in
// opposite directions, would wait for both in turn: 32 x 2048 x 512 109 -> 127 us.  It composes a tile's maps around one
// barrier.)  A slot is written for the next tile only after the wave that reads it has sent on what it read.  All waves
// of a workgroup are resident, so every wait ends.
template <typename P>
struct Relay {
  float slot[P::WAVES][P::SLAB];
  uint32_t tag[P::WAVES];
};
template <typename P, int VEC = P::VEC>
__device__ __forceinline__ void relay_put(const P& at, Relay<P>& relay, int wave, uint32_t tag, const float (&c)[VEC]) {
  if (at.lane < P::CT) put_lds<VEC>(&relay.slot[wave][at.ct * VEC], c);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  if (at.lane == 0) __hip_atomic_store(&relay.tag[wave], tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
template <typename P, int VEC = P::VEC>
__device__ __forceinline__ void relay_get(const P& at, Relay<P>& relay, uint32_t tag, float (&c)[VEC]) {
  while (__hip_atomic_load(&relay.tag[at.wave], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) != tag) {
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  const Vec<float, VEC> v = get_lds<VEC>(&relay.slot[at.wave][at.ct * VEC]);
#pragma unroll
  for (int j = 0; j < VEC; ++j) c[j] = v.v[j];
}
// One wave's part of a tile: takes the carry, gives the next wave what the map (A, B) of its own steps makes of it (the
// last wave gives it to the next tile's first), and returns what a thread starts from, by its map (pa, pb).
template <typename P, int VEC = P::VEC>
__device__ __forceinline__ void relay_pass(const P& at, Relay<P>& relay, uint32_t round, const float (&A)[VEC],
                                           const float (&B)[VEC], const float (&pa)[VEC], const float (&pb)[VEC],
                                           float (&carry)[VEC], float (&mine)[VEC]) {
  relay_get(at, relay, round, carry);
  float after[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    after[j] = fmaf(A[j], carry[j], B[j]);
    mine[j] = fmaf(pa[j], carry[j], pb[j]);
  }
  if (at.wave + 1 < P::WAVES)
    relay_put(at, relay, at.wave + 1, round, after);
  else
    relay_put(at, relay, 0, round + 1, after);
}
// Empties the relay (all threads; a barrier follows).
template <typename P>
__device__ __forceinline__ void relay_clear(Relay<P>& relay) {
  if (threadIdx.x < P::WAVES) relay.tag[threadIdx.x] = 0;
}

// The carry at a segment's start: the maps of the n segments before it, segment `first` + i `step` for i = 0 .. n - 1 in
// this order, applied to `carry`.  Each time group composes a run of them, and the runs are composed as a tile's are.
// (One thread after the other through the same maps, an L2 latency each, took 60 us for 255 segments.)
template <typename T, typename P, int SUMS, int VEC = P::VEC>
__device__ __forceinline__ void fold_segments(const ScanArgs<T>& p, const P& at, int first, int step, int n,
                                              TileMaps<P, SUMS>& lds, float (&carry)[VEC]) {
  if (n == 0) return;
  float A[VEC], B[1][VEC], pa[1][VEC], pb[1][VEC], none[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[0][j] = 0.0f;
  if (at.on) {
    const int run = (n + P::TG - 1) / P::TG, end = min(n, (at.tg + 1) * run);
#pragma unroll 4
    for (int i = at.tg * run; i < end; ++i) {
      const int64_t o = (int64_t)(first + i * step) * p.channels + at.n;
      const Vec<float, VEC> a = load_vec<float, VEC>(p.seg_a + o), b = load_vec<float, VEC>(p.seg_b + o);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        B[0][j] = fmaf(a.v[j], B[0][j], b.v[j]);
        A[j] *= a.v[j];
      }
    }
    hold_factors(A);
  }
  wave_maps<P, 1, false>(at.lane, A, B, pa, pb);
  if (at.lane < P::CT) {
    put_lds<VEC>(&lds[at.wave][0][at.ct * VEC], A);
    put_lds<VEC>(&lds[at.wave][1][at.ct * VEC], B[0]);
  }
  lds_barrier();
  fold_waves<P, SUMS, 0, false>(at, lds, pa[0], pb[0], carry, none);
}

// A thread's rows of a tile.  Steps past the row's length hold f = +inf, so that a = 1 and 1 - a = 0 without a test,
// and zeros.
template <typename T, typename P, bool G, bool O, bool D>
struct Rows {
  static constexpr int VEC = P::VEC, R = P::R;
  Vec<T, VEC> f[R], g[R], o[R], d[R];

  __device__ __forceinline__ void load(const ScanArgs<T>& p, const P& at, int tile) {
    const int t0 = tile * P::TILE + at.tg * R;
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

// Zeros for the tiles first .. end - 1, which no row of the slab reaches, of dst [B][T][PARTS H].
template <int PARTS, typename P, typename T>
__device__ __forceinline__ void zero_tiles(T* dst, const ScanArgs<T>& p, const P& at, int first, int end) {
  if (!at.on) return;
  const Vec<T, P::VEC> zero = {};
  const int t_end = min(end * P::TILE, p.T_);
  for (int t = first * P::TILE + at.tg; t < t_end; t += P::TG) {
    T* const q = dst + (at.b * p.T_ + t) * (int64_t)(PARTS * p.H) + at.h;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) store_vec(q + k * p.H, zero);
  }
}

template <typename P, int VEC = P::VEC>
__device__ __forceinline__ void load_carry(const float* src, const P& at, float (&c)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) c[j] = 0.0f;
  if (!src || !at.on) return;
  const Vec<float, VEC> v = load_vec<float, VEC>(src + at.n);
#pragma unroll
  for (int j = 0; j < VEC; ++j) c[j] = v.v[j];
}

template <typename P, int VEC = P::VEC>
__device__ __forceinline__ void store_carry(float* dst, const P& at, const float (&c)[VEC]) {
  Vec<float, VEC> v;
#pragma unroll
  for (int j = 0; j < VEC; ++j) v.v[j] = c[j];
  store_vec(dst + at.n, v);
}

// The maps of the segments, for the launch that follows: of all but the last in order (of c), or of all but the first
// in reverse order (of E).  Each time group composes a run of the segment, and the runs are composed once at the end.
template <typename T, typename P, bool REVERSE, bool GATED>
__global__ void __launch_bounds__(P::THREADS) scan_maps_kernel(ScanArgs<T> p) {
  constexpr int VEC = P::VEC, R = P::R;
  __shared__ alignas(16) TileMaps<P, 1> lds;
  const int seg = blockIdx.x / p.slabs + (REVERSE ? 1 : 0);
  const P at(p, slab_of(blockIdx.x % p.slabs, p.slabs));
  float A[VEC], B[1][VEC], pa[1][VEC], pb[1][VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[0][j] = 0.0f;
  const int run = p.seg_tiles * R, first = seg * p.seg_tiles * P::TILE + at.tg * run;
  const int steps = min(run, at.len - first);
  const T* const src = p.gates + at.b * p.stride_b + (int64_t)first * p.stride_t + at.h;
  const T* const grad = REVERSE ? p.d_out + (at.b * p.T_ + first) * (int64_t)p.H + at.h : nullptr;
  const auto rows = [&](int t0, auto count) __attribute__((always_inline)) {
    constexpr int N = decltype(count)::value;
    Vec<T, VEC> f[N], x[N], o[N];  // x: g, or the gradient of the output
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const T* const q = src + (int64_t)(t0 + r) * p.stride_t;
      f[r] = load_vec<T, VEC>(q);
      x[r] = load_vec<T, VEC>(REVERSE ? grad + (int64_t)(t0 + r) * p.H : q + p.H);
      if (REVERSE && GATED) o[r] = load_vec<T, VEC>(q + 2 * p.H);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = REVERSE ? N - 1 - i : i;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float s, ns;
        logistic((float)f[r].v[j], s, ns);
        float v = (float)x[r].v[j];
        if (REVERSE) {
          if (GATED) v *= sigmoid((float)o[r].v[j]);
          B[0][j] = s * (B[0][j] + v);
        } else {
          B[0][j] = fmaf(s, B[0][j], ns * v);
        }
        A[j] *= s;
      }
    }
  };
  using Many = std::integral_constant<int, 4>;
  using One = std::integral_constant<int, 1>;
  if (REVERSE) {
    int t = steps;
    for (; t % 4 != 0 && t > 0; --t) rows(t - 1, One());
    for (; t > 0; t -= 4) rows(t - 4, Many());
  } else {
    int t = 0;
    for (; t + 4 <= steps; t += 4) rows(t, Many());
    for (; t < steps; ++t) rows(t, One());
  }
  hold_factors(A);
  wave_maps<P, 1, REVERSE>(at.lane, A, B, pa, pb);
  put_maps<P, 1>(at, lds, A, B);
  lds_barrier();
  if (!at.on || at.tg != 0) return;
  float prod[VEC], sum[VEC], none[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) prod[j] = 1.0f, sum[j] = 0.0f;
#pragma unroll
  for (int w = 0; w < P::WAVES; ++w) {
    const Vec<float, VEC> a = get_lds<VEC>(&lds[w][0][at.ct * VEC]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) prod[j] *= a.v[j];
  }
  hold_factors(prod);
  fold_waves<P, 1, 0, REVERSE>(at, lds, pa[0], pb[0], sum, none);
  store_carry(p.seg_a + (int64_t)seg * p.channels, at, prod);
  store_carry(p.seg_b + (int64_t)seg * p.channels, at, sum);
}

template <typename T, typename P, bool GATED>
__global__ void __launch_bounds__(P::THREADS, sizeof(T) == 2 ? 4 : 1) scan_forward_kernel(ScanArgs<T> p) {
  constexpr int VEC = P::VEC, R = P::R;
  __shared__ alignas(16) TileMaps<P, 1> lds;
  __shared__ alignas(16) Relay<P> relay;
  const int seg = blockIdx.x / p.slabs;
  const P at(p, slab_of(blockIdx.x % p.slabs, p.slabs));
  float carry[VEC];
  load_carry(p.c0, at, carry);
  const int tile_first = seg * p.seg_tiles, tile_end = min(p.tiles, (seg + 1) * p.seg_tiles);
  fold_segments<T, P, 1>(p, at, 0, 1, seg, lds, carry);
  relay_clear(relay);
  lds_barrier();
  if (at.wave == 0) relay_put(at, relay, 0, 1, carry);
  uint32_t round = 0;
  using Tile = Rows<T, P, true, GATED, false>;
  const auto process = [&](const Tile& x, int tile) __attribute__((always_inline)) {
    const int t0 = tile * P::TILE + at.tg * R;
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
    hold_factors(A);
    wave_maps<P, 1, false>(at.lane, A, B, pa, pb);
    float c[VEC];
    relay_pass(at, relay, ++round, A, B[0], pa[0], pb[0], carry, c);
    if (p.states && at.on && at.tg == 0) store_carry(p.states + (int64_t)tile * p.channels, at, carry);
    if (!at.on) return;
    T* dst = p.out + (at.b * p.T_ + t0) * (int64_t)p.H + at.h;
    Vec<T, VEC> y[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float h[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        c[j] = fmaf(a[r][j], c[j], b[r][j]);
        h[j] = GATED ? c[j] * sigmoid((float)x.o[r].v[j]) : c[j];
      }
      y[r] = round_to<T, VEC>(h);
    }
    if (__all(t0 + R <= at.len)) {
#pragma unroll
      for (int r = 0; r < R; ++r) store_vec(dst + (int64_t)r * p.H, y[r]);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (t0 + r < p.T_) store_vec(dst + (int64_t)r * p.H, zero_unless(t0 + r < at.len, y[r]));
    }
  };
  const int live_end = min(tile_end, at.live_tiles);
  Tile x, next;  // a tile's loads are in flight while the one before is computed
  if (tile_first < live_end) next.load(p, at, tile_first);
  for (int tile = tile_first; tile < live_end; ++tile) {
    x = next;
    if (P::MANY && tile + 1 < live_end) next.load(p, at, tile + 1);
    process(x, tile);
  }
  zero_tiles<1>(p.out, p, at, max(tile_first, live_end), tile_end);
  if (at.wave == 0) {
    relay_get(at, relay, round + 1, carry);
    if (at.on && at.tg == 0 && seg == p.segs - 1 && p.c_n) store_carry(p.c_n, at, carry);
  }
}

// Backward: tiles from the last to the first.  With an output gate 236 to 254 registers for 16-bit elements, two waves per
// SIMD, and 256 and 16 accumulation registers for 32-bit ones, one wave.  Either moves its bytes at the copy's rate
// (5.2 TB/s): 16 x 4096 x 2048 bf16 353 us, at that rate 361; 16 x 2048 x 2048 fp32 365 and 361.
template <typename T, typename P, bool GATED>
__global__ void __launch_bounds__(P::THREADS) scan_backward_kernel(ScanArgs<T> p) {
  constexpr int VEC = P::VEC, R = P::R;
  constexpr int kParts = GATED ? 3 : 2;
  __shared__ alignas(16) WaveMaps<P, 2> lds;
  const int seg = blockIdx.x / p.slabs;
  const P at(p, slab_of(blockIdx.x % p.slabs, p.slabs));
  float carry[VEC];
  load_carry(p.d_cn, at, carry);
  const int tile_first = seg * p.seg_tiles, tile_last = min(p.tiles, (seg + 1) * p.seg_tiles) - 1;
  const int live_last = min(tile_last, at.live_tiles - 1);
  // in the half that the first tile, live_last, does not write: no barrier follows
  fold_segments<T, P, 2>(p, at, p.segs - 1, -1, p.segs - 1 - seg, lds[(live_last + 1) & 1], carry);
  struct Tile : Rows<T, P, true, GATED, true> {
    float start[VEC];  // c before the tile, from the forward pass
    __device__ __forceinline__ void load(const ScanArgs<T>& p, const P& at, int tile) {
      Rows<T, P, true, GATED, true>::load(p, at, tile);
      load_carry(p.states + (int64_t)tile * p.channels, at, start);
    }
  };
  const auto process = [&](const Tile& x, int tile) __attribute__((always_inline)) {
    const int t0 = tile * P::TILE + at.tg * R;
    float a[R][VEC], na[R][VEC], u[R][VEC], w[R][VEC];  // a, 1 - a, u = s dh, w = (1 - s) u
    float A[VEC], B[2][VEC], pa[2][VEC], pb[2][VEC];    // sums in order (for c) and in reverse order (for E)
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[0][j] = B[1][j] = 0.0f;
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
        B[1][j] = a[r][j] * (B[1][j] + u[r][j]);
        A[j] *= a[r][j];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < VEC; ++j) B[0][j] = fmaf(a[r][j], B[0][j], na[r][j] * (float)x.g[r].v[j]);
    hold_factors(A);
    wave_maps<P, 2, false>(at.lane, A, B, pa, pb);
    auto& maps = lds[tile & 1];
    put_maps<P, 2>(at, maps, A, B);
    lds_barrier();
    float e[VEC], start[VEC], c[VEC], before[R][VEC];
    fold_waves<P, 2, 1, true>(at, maps, pa[1], pb[1], carry, e);
    if (!at.on) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) start[j] = x.start[j];
    fold_waves<P, 2, 0, false>(at, maps, pa[0], pb[0], start, c);
    Vec<T, VEC> df[R], dg[R], d_o[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float d[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        before[r][j] = c[j];
        c[j] = fmaf(a[r][j], c[j], na[r][j] * (float)x.g[r].v[j]);
        d[j] = GATED ? w[r][j] * c[j] : 0.0f;
      }
      if (GATED) d_o[r] = round_to<T, VEC>(d);
    }
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      float n[VEC], m[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float D = u[r][j] + e[j];
        n[j] = na[r][j] * D;
        e[j] = a[r][j] * D;
        m[j] = a[r][j] * n[j] * (before[r][j] - (float)x.g[r].v[j]);
      }
      dg[r] = round_to<T, VEC>(n);
      df[r] = round_to<T, VEC>(m);
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
  };
  zero_tiles<kParts>(p.d_gates, p, at, max(tile_first, at.live_tiles), tile_last + 1);
  Tile x, next;  // (as in the forward kernel)
  if (live_last >= tile_first) next.load(p, at, live_last);
  for (int tile = live_last; tile >= tile_first; --tile) {
    x = next;
    if (P::MANY && tile > tile_first) next.load(p, at, tile - 1);
    process(x, tile);
  }
  if (at.on && at.tg == 0 && seg == 0 && p.d_c0) store_carry(p.d_c0, at, carry);
}

// ---- a few steps ----
// One step (serving) or up to eight: a thread carries VEC channels through them one after the other, nothing to scan.
// In tiles of 16 steps and here, forward / backward us: 199 x 5 x 2048 bf16 9.9 / 15.4 and 7.7 / 8.8, 2000 x 8 x 256
// 11.5 / 18.8 and 10.5 / 12.3, 400 x 8 x 400 fp32 7.0 / 11.1 and 7.4 / 9.3.  With more steps the chain of loads takes
// over: 300 x 16 x 512 bf16 forward 7.3 and 13.9.
constexpr int kShort = 8;
constexpr int kShortThreads = 256;

// A thread's channels: f(integral constant N, b, h) for N of them from h on.  A row's last piece goes one channel at a
// time where it is not full: c_n may be c0, so that no channel may be another thread's too.
template <int VEC, typename T, typename F>
__device__ __forceinline__ void short_pieces(const ScanArgs<T>& p, F&& f) {
  const uint32_t piece = blockIdx.x * kShortThreads + threadIdx.x, per = (p.H + VEC - 1) / VEC;
  if (piece >= p.pieces) return;
  const int64_t b = piece / per;
  const int h = (int)(piece % per) * VEC;
  if (h + VEC <= p.H) {
    f(std::integral_constant<int, VEC>(), b, h);
  } else {
    for (int k = h; k < p.H; ++k) f(std::integral_constant<int, 1>(), b, k);
  }
}

template <typename T, int VEC, bool GATED>
__global__ void __launch_bounds__(kShortThreads) scan_forward_short_kernel(ScanArgs<T> p) {
  short_pieces<VEC>(p, [&](auto width, int64_t b, int h) __attribute__((always_inline)) {
    constexpr int N = decltype(width)::value, U = 4;  // U steps are loaded at a time
    const int len = p.lengths ? min(max(p.lengths[b], 0), p.T_) : p.T_;
    const int64_t n = b * p.H + h;
    Vec<float, N> c = {};
    if (p.c0) c = load_vec<float, N>(p.c0 + n);
    if (p.states) store_vec(p.states + n, c);
    const T* src = p.gates + b * p.stride_b + h;
    T* dst = p.out + b * p.T_ * p.H + h;
    for (int t = 0; t < p.T_; t += U) {
      Vec<T, N> f[U] = {}, g[U] = {}, o[U] = {};
#pragma unroll
      for (int r = 0; r < U; ++r) {
        if (t + r < len) {
          f[r] = load_vec<T, N>(src), g[r] = load_vec<T, N>(src + p.H);
          if (GATED) o[r] = load_vec<T, N>(src + 2 * p.H);
        }
        src += p.stride_t;
      }
#pragma unroll
      for (int r = 0; r < U; ++r) {
        if (t + r < p.T_) {
          float y[N];
#pragma unroll
          for (int j = 0; j < N; ++j) {
            float a, na;
            logistic((float)f[r].v[j], a, na);
            const float next = fmaf(a, c.v[j], na * (float)g[r].v[j]);
            c.v[j] = t + r < len ? next : c.v[j];
            y[j] = GATED ? next * sigmoid((float)o[r].v[j]) : next;
          }
          store_vec(dst, zero_unless(t + r < len, round_to<T, N>(y)));
        }
        dst += p.H;
      }
    }
    if (p.c_n) store_vec(p.c_n + n, c);
  });
}

template <typename T, int VEC, bool GATED>
__global__ void __launch_bounds__(kShortThreads) scan_backward_short_kernel(ScanArgs<T> p) {
  short_pieces<VEC>(p, [&](auto width, int64_t b, int h) __attribute__((always_inline)) {
    constexpr int N = decltype(width)::value, R = kShort, kParts = GATED ? 3 : 2;
    const int len = p.lengths ? min(max(p.lengths[b], 0), p.T_) : p.T_;
    const int64_t n = b * p.H + h;
    Vec<T, N> f[R] = {}, g[R] = {}, o[R] = {}, d[R] = {};
    const T* src = p.gates + b * p.stride_b + h;
    const T* grad = p.d_out + b * p.T_ * p.H + h;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < len) {
        f[r] = load_vec<T, N>(src), g[r] = load_vec<T, N>(src + p.H);
        if (GATED) o[r] = load_vec<T, N>(src + 2 * p.H);
        d[r] = load_vec<T, N>(grad);
      }
      src += p.stride_t, grad += p.H;
    }
    Vec<float, N> c = load_vec<float, N>(p.states + n), e = {};
    if (p.d_cn) e = load_vec<float, N>(p.d_cn + n);
    float before[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float a, na;
        logistic((float)f[r].v[j], a, na);
        before[r][j] = c.v[j];
        c.v[j] = fmaf(a, c.v[j], na * (float)g[r].v[j]);  // (past the row's end it is not used)
      }
    }
    T* const dst = p.d_gates + b * p.T_ * (kParts * p.H) + h;
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      if (r >= p.T_) continue;
      const bool live = r < len;
      float df[N], dg[N], d_o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float a, na, u = (float)d[r].v[j];
        const float gv = (float)g[r].v[j];
        logistic((float)f[r].v[j], a, na);
        if (GATED) {
          float s, ns;
          logistic_fast((float)o[r].v[j], s, ns);
          u *= s;
          d_o[j] = ns * u * fmaf(a, before[r][j], na * gv);
        }
        const float D = u + e.v[j], k = na * D;
        if (live) e.v[j] = a * D;
        dg[j] = k;
        df[j] = a * k * (before[r][j] - gv);
      }
      T* const q = dst + (int64_t)r * (kParts * p.H);
      store_vec(q, zero_unless(live, round_to<T, N>(df)));
      store_vec(q + p.H, zero_unless(live, round_to<T, N>(dg)));
      if (GATED) store_vec(q + 2 * p.H, zero_unless(live, round_to<T, N>(d_o)));
    }
    if (p.d_c0) store_vec(p.d_c0 + n, e);
  });
}

template <typename T, typename P, bool GATED, bool BACKWARD>
hipError_t launch_slabs(const ScanArgs<T>& p, hipStream_t s) {
  const dim3 block(P::THREADS);
  if constexpr (P::MANY) {
    if (p.segs > 1) {
      hipLaunchKernelGGL((scan_maps_kernel<T, P, BACKWARD, BACKWARD && GATED>),
                         dim3(p.slabs * (unsigned)(p.segs - 1)), block, 0, s, p);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  const dim3 grid(p.slabs * (unsigned)p.segs);
  if constexpr (BACKWARD)
    hipLaunchKernelGGL((scan_backward_kernel<T, P, GATED>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((scan_forward_kernel<T, P, GATED>), grid, block, 0, s, p);
  return hipGetLastError();
}

template <typename T, int VEC, bool GATED, bool BACKWARD>
hipError_t launch_vec(const ScanArgs<T>& p, hipStream_t s) {
  if (p.T_ >= 1 && p.T_ <= kShort) {
    const dim3 grid((p.pieces + kShortThreads - 1) / kShortThreads), block(kShortThreads);
    if constexpr (BACKWARD)
      hipLaunchKernelGGL((scan_backward_short_kernel<T, VEC, GATED>), grid, block, 0, s, p);
    else
      hipLaunchKernelGGL((scan_forward_short_kernel<T, VEC, GATED>), grid, block, 0, s, p);
    return hipGetLastError();
  }
  if constexpr (VEC == 1) {
    return launch_slabs<T, Narrow, GATED, BACKWARD>(p, s);
  } else {
    if (p.T_ <= Steps16::TILE) return launch_slabs<T, Steps16, GATED, BACKWARD>(p, s);
    if (p.T_ <= Steps32::TILE) return launch_slabs<T, Steps32, GATED, BACKWARD>(p, s);
    if (p.T_ <= Steps64::TILE) return launch_slabs<T, Steps64, GATED, BACKWARD>(p, s);
    if constexpr (sizeof(T) == 2)
      if (p.ct == Wide::CT) return launch_slabs<T, Wide, GATED, BACKWARD>(p, s);
    return launch_slabs<T, Usual, GATED, BACKWARD>(p, s);
  }
}

template <typename T, bool BACKWARD>
hipError_t launch_scan(const ScanArgs<T>& p, bool gated, hipStream_t s) {
  const auto go = [&](auto vec) {
    constexpr int V = decltype(vec)::value;
    return gated ? launch_vec<T, V, true, BACKWARD>(p, s) : launch_vec<T, V, false, BACKWARD>(p, s);
  };
  return scan_vec(p.H) == 4 ? go(std::integral_constant<int, 4>()) : go(std::integral_constant<int, 1>());
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
  if (!aligned(workspace, 16)) return op_error(PLH_ERR_INVALID, what, "workspace must be 16-byte aligned");
  return PLH_OK;
}

template <typename T>
ScanArgs<T> scan_args(const void* gates, int64_t stride_b, int64_t stride_t, int64_t batch, int64_t seq_len, int hidden,
                      const int32_t* lengths, void* workspace, bool backward) {
  const Layout l = layout_for(sizeof(T), batch, seq_len, hidden, backward);
  ScanArgs<T> p = {};
  p.gates = (const T*)gates;
  p.stride_b = stride_b, p.stride_t = stride_t;
  p.channels = batch * hidden;
  p.T_ = (int)seq_len, p.H = hidden;
  p.tiles = l.tiles, p.seg_tiles = l.seg_tiles, p.segs = l.segs;
  p.slabs = (unsigned)l.slabs, p.ct = l.ct;
  p.pieces = (unsigned)pieces_of(batch, hidden);
  p.lengths = lengths;
  p.seg_a = (float*)workspace;
  p.seg_b = p.seg_a ? p.seg_a + (p.channels * l.segs + 3) / 4 * 4 : nullptr;
  return p;
}

}  // namespace
}  // namespace plh

extern "C" {

int64_t plh_gated_scan_states(int64_t seq_len) { return seq_len < 0 ? -1 : (seq_len + plh::kTile - 1) / plh::kTile; }

int64_t plh_gated_scan_workspace_bytes(int64_t batch, int64_t seq_len, int hidden) {
  if (batch < 0 || seq_len < 0 || hidden < 1 || seq_len > (1 << 30) || batch > (1 << 29)) return -1;
  int segs = 1;  // the most of any type, in either direction
  for (int elem : {2, 4})
    for (bool backward : {false, true})
      segs = std::max(segs, plh::layout_for(elem, batch, seq_len, hidden, backward).segs);
  if (segs <= 1) return 0;
  return 2 * ((batch * hidden * segs + 3) / 4 * 4) * (int64_t)sizeof(float);
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
    auto p = plh::scan_args<T>(gates, stride_b, stride_t, batch, seq_len, hidden, lengths, workspace, false);
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
    auto p = plh::scan_args<T>(gates, stride_b, stride_t, batch, seq_len, hidden, lengths, workspace, true);
    p.states = const_cast<float*>(states), p.d_out = (const T*)d_out, p.d_cn = d_cn;
    p.d_gates = (T*)d_gates, p.d_c0 = d_c0;
    e = plh::launch_scan<T, true>(p, output_gate != 0, (hipStream_t)stream);
  });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

}  // extern "C"
