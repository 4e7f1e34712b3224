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
constexpr int kScanGroups = 2048;

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
    lane = tid % kWave, wave = tid / kWave, ct = tid % CT, tg = tid / CT;
    n = (int64_t)slab * kSlab + ct * VEC;
    on = n < p.channels;
    b = 0, h = 0, len = 0;
    if (on) {
      if (p.channels <= 0xFFFFFFFFll) {
        b = (uint32_t)n / (uint32_t)p.H;
        h = (int)((uint32_t)n % (uint32_t)p.H);
      } else {
        b = n / p.H;
        h = (int)(n % p.H);
      }
      len = p.T_;
      if (p.lengths) len = min(max(p.lengths[b], 0), p.T_);
    }
  }
};

// The maps of the time groups, composed: on entry A, B are a thread's own map (FORWARD: of its steps in order,
// else in reverse order); on return the map of everything in this wave that comes before this thread's steps, with the
// whole wave's map in LDS at [wave][channel] for the caller to fold after a barrier.
template <int VEC, bool FORWARD>
__device__ __forceinline__ void wave_maps(const Place<VEC>& at, float (&A)[VEC], float (&B)[VEC],
                                          float (*lds_a)[kSlab], float (*lds_b)[kSlab]) {
  constexpr int CT = Place<VEC>::CT;
#pragma unroll
  for (int d = CT; d < kWave; d *= 2) {
    const bool has = FORWARD ? at.lane >= d : at.lane < kWave - d;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float pa = FORWARD ? __shfl_up(A[j], d) : __shfl_down(A[j], d);
      const float pb = FORWARD ? __shfl_up(B[j], d) : __shfl_down(B[j], d);
      if (has) {
        B[j] = fmaf(A[j], pb, B[j]);
        A[j] *= pa;
      }
    }
  }
  const bool whole = FORWARD ? at.lane >= kWave - CT : at.lane < CT;
  if (whole) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      lds_a[at.wave][at.ct * VEC + j] = A[j];
      lds_b[at.wave][at.ct * VEC + j] = B[j];
    }
  }
  const bool first = FORWARD ? at.lane < CT : at.lane >= kWave - CT;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float pa = FORWARD ? __shfl_up(A[j], CT) : __shfl_down(A[j], CT);
    const float pb = FORWARD ? __shfl_up(B[j], CT) : __shfl_down(B[j], CT);
    A[j] = first ? 1.0f : pa;
    B[j] = first ? 0.0f : pb;
  }
}

// The carry through the four waves' maps: `carry` becomes the value after the whole tile, and the return in `mine` is
// the value that this thread's steps start from.  (A, B) is the thread's map from wave_maps.
template <int VEC, bool FORWARD>
__device__ __forceinline__ void fold_waves(const Place<VEC>& at, const float (&A)[VEC], const float (&B)[VEC],
                                           const float (*lds_a)[kSlab], const float (*lds_b)[kSlab],
                                           float (&carry)[VEC], float (&mine)[VEC]) {
  constexpr int W = kScanThreads / kWave;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int w = FORWARD ? i : W - 1 - i;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (w == at.wave) mine[j] = fmaf(A[j], carry[j], B[j]);
      carry[j] = fmaf(lds_a[w][at.ct * VEC + j], carry[j], lds_b[w][at.ct * VEC + j]);
    }
  }
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

// Forward.  MAPS: only the segments' maps (of all but the last), for the launch that follows.
template <typename T, int VEC, bool GATED, bool MAPS>
__global__ void __launch_bounds__(kScanThreads) scan_forward_kernel(ScanArgs<T> p) {
  using P = Place<VEC>;
  constexpr int R = P::R;
  __shared__ float lds_a[2][4][kSlab], lds_b[2][4][kSlab];
  const unsigned slab = blockIdx.x % p.slabs;
  const int seg = blockIdx.x / p.slabs;
  const P at(p, slab);
  float carry[VEC], prod[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) carry[j] = 0.0f, prod[j] = 1.0f;
  if (!MAPS && at.on) {
    if (p.c0) {
      const Vec<float, VEC> c = load_vec<float, VEC>(p.c0 + at.n);
#pragma unroll
      for (int j = 0; j < VEC; ++j) carry[j] = c.v[j];
    }
    fold_segments<T, VEC>(p, at, 0, seg, 1, carry);
  }
  const int tile_end = min(p.tiles, (seg + 1) * p.seg_tiles);
  const T* const row = p.gates + at.b * p.stride_b + at.h;
  for (int tile = seg * p.seg_tiles; tile < tile_end; ++tile) {
    const int t0 = tile * kTile + at.tg * R;
    Vec<T, VEC> f[R] = {}, g[R] = {}, o[R] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (t0 + r < at.len) {
        const T* src = row + (int64_t)(t0 + r) * p.stride_t;
        f[r] = load_vec<T, VEC>(src);
        g[r] = load_vec<T, VEC>(src + p.H);
        if (GATED && !MAPS) o[r] = load_vec<T, VEC>(src + 2 * p.H);
      }
    }
    float a[R][VEC], b[R][VEC], A[VEC], B[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = t0 + r < at.len;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float s = 1.0f, ns = 0.0f, in = 0.0f;
        if (live) {
          logistic((float)f[r].v[j], s, ns);
          in = ns * (float)g[r].v[j];
        }
        a[r][j] = s, b[r][j] = in;
        B[j] = fmaf(s, B[j], in);
        A[j] *= s;
      }
    }
    float(*la)[kSlab] = lds_a[tile & 1];
    float(*lb)[kSlab] = lds_b[tile & 1];
    wave_maps<VEC, true>(at, A, B, la, lb);
    __syncthreads();  // (the other half of the buffers is written next, so one barrier per tile is enough)
    if (!MAPS && p.states && at.on && at.tg == 0) {
      Vec<float, VEC> c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) c.v[j] = carry[j];
      store_vec(p.states + (int64_t)tile * p.channels + at.n, c);
    }
    float c[VEC];
    if (MAPS) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < VEC; ++j) prod[j] *= la[w][at.ct * VEC + j];
    }
    fold_waves<VEC, true>(at, A, B, la, lb, carry, c);
    if (!MAPS && at.on) {
      T* dst = p.out + (at.b * p.T_ + t0) * (int64_t)p.H + at.h;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (t0 + r < p.T_) {
          Vec<T, VEC> y;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            c[j] = fmaf(a[r][j], c[j], b[r][j]);
            float h = c[j];
            if (GATED) {
              float s, ns;
              logistic((float)o[r].v[j], s, ns);
              h *= s;
            }
            y.v[j] = (T)(t0 + r < at.len ? h : 0.0f);
          }
          store_vec(dst + (int64_t)r * p.H, y);
        }
      }
    }
  }
  if (at.on && at.tg == 0) {
    Vec<float, VEC> va, vb;
#pragma unroll
    for (int j = 0; j < VEC; ++j) va.v[j] = prod[j], vb.v[j] = carry[j];
    if (MAPS) {
      store_vec(p.seg_a + (int64_t)seg * p.channels + at.n, va);
      store_vec(p.seg_b + (int64_t)seg * p.channels + at.n, vb);
    } else if (seg == p.segs - 1 && p.c_n) {
      store_vec(p.c_n + at.n, vb);
    }
  }
}

// Backward: tiles from the last to the first.  MAPS: only the segments' maps of E (of all but the first).
template <typename T, int VEC, bool GATED, bool MAPS>
__global__ void __launch_bounds__(kScanThreads) scan_backward_kernel(ScanArgs<T> p) {
  using P = Place<VEC>;
  constexpr int R = P::R;
  constexpr int kParts = GATED ? 3 : 2;
  __shared__ float lds_a[2][4][kSlab], lds_b[2][4][kSlab], lds_fa[2][4][kSlab], lds_fb[2][4][kSlab];
  const unsigned slab = blockIdx.x % p.slabs;
  const int seg = blockIdx.x / p.slabs + (MAPS ? 1 : 0);
  const P at(p, slab);
  float carry[VEC], prod[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) carry[j] = 0.0f, prod[j] = 1.0f;
  if (!MAPS && at.on) {
    if (p.d_cn) {
      const Vec<float, VEC> c = load_vec<float, VEC>(p.d_cn + at.n);
#pragma unroll
      for (int j = 0; j < VEC; ++j) carry[j] = c.v[j];
    }
    fold_segments<T, VEC>(p, at, p.segs - 1, seg, -1, carry);
  }
  const int tile_first = seg * p.seg_tiles;
  const T* const row = p.gates + at.b * p.stride_b + at.h;
  for (int tile = min(p.tiles, (seg + 1) * p.seg_tiles) - 1; tile >= tile_first; --tile) {
    const int t0 = tile * kTile + at.tg * R;
    Vec<T, VEC> f[R] = {}, g[R] = {}, o[R] = {}, dh[R] = {};
    const T* const d_row = p.d_out + (at.b * p.T_ + t0) * (int64_t)p.H + at.h;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (t0 + r < at.len) {
        const T* src = row + (int64_t)(t0 + r) * p.stride_t;
        f[r] = load_vec<T, VEC>(src);
        if (!MAPS) g[r] = load_vec<T, VEC>(src + p.H);
        if (GATED) o[r] = load_vec<T, VEC>(src + 2 * p.H);
        dh[r] = load_vec<T, VEC>(d_row + (int64_t)r * p.H);
      }
    }
    float a[R][VEC], na[R][VEC], u[R][VEC], A[VEC], E[VEC], FA[VEC], FB[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, E[j] = 0.0f, FB[j] = 0.0f;
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      const bool live = t0 + r < at.len;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float s = 1.0f, ns = 0.0f, d = 0.0f;
        if (live) {
          logistic((float)f[r].v[j], s, ns);
          d = (float)dh[r].v[j];
          if (GATED) {
            float so, nso;
            logistic((float)o[r].v[j], so, nso);
            d *= so;
          }
        }
        a[r][j] = s, na[r][j] = ns, u[r][j] = d;
        E[j] = s * (E[j] + d);
        A[j] *= s;
      }
    }
    const int half = tile & 1;
    if (!MAPS) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float in = t0 + r < at.len ? na[r][j] * (float)g[r].v[j] : 0.0f;
          FB[j] = fmaf(a[r][j], FB[j], in);
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) FA[j] = A[j];
      wave_maps<VEC, true>(at, FA, FB, lds_fa[half], lds_fb[half]);
    }
    wave_maps<VEC, false>(at, A, E, lds_a[half], lds_b[half]);
    __syncthreads();  // (as in the forward kernel)
    if (MAPS) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < VEC; ++j) prod[j] *= lds_a[half][w][at.ct * VEC + j];
    }
    float e[VEC];
    fold_waves<VEC, false>(at, A, E, lds_a[half], lds_b[half], carry, e);
    if (!MAPS && at.on) {
      // c before each of this thread's steps, from the state that the forward pass left at the tile's start
      const Vec<float, VEC> st = load_vec<float, VEC>(p.states + (int64_t)tile * p.channels + at.n);
      float start[VEC], c[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) start[j] = st.v[j];
      fold_waves<VEC, true>(at, FA, FB, lds_fa[half], lds_fb[half], start, c);
      float before[R][VEC];
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          before[r][j] = c[j];
          const float in = t0 + r < at.len ? na[r][j] * (float)g[r].v[j] : 0.0f;
          c[j] = fmaf(a[r][j], c[j], in);
        }
      }
      T* const dst = p.d_gates + (at.b * p.T_ + t0) * (int64_t)(kParts * p.H) + at.h;
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
        const bool live = t0 + r < at.len;
        Vec<T, VEC> df, dg, d_o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float D = u[r][j] + e[j];
          e[j] = a[r][j] * D;
          df.v[j] = dg.v[j] = d_o.v[j] = (T)0.0f;
          if (live) {
            const float gv = (float)g[r].v[j];
            dg.v[j] = (T)(na[r][j] * D);
            df.v[j] = (T)(e[j] * na[r][j] * (before[r][j] - gv));
            if (GATED) {
              float so, nso;
              logistic((float)o[r].v[j], so, nso);
              d_o.v[j] = (T)(nso * u[r][j] * fmaf(a[r][j], before[r][j], na[r][j] * gv));
            }
          }
        }
        if (t0 + r < p.T_) {
          T* q = dst + (int64_t)r * (kParts * p.H);
          store_vec(q, df);
          store_vec(q + p.H, dg);
          if (GATED) store_vec(q + 2 * p.H, d_o);
        }
      }
    }
  }
  if (at.on && at.tg == 0) {
    Vec<float, VEC> va, vb;
#pragma unroll
    for (int j = 0; j < VEC; ++j) va.v[j] = prod[j], vb.v[j] = carry[j];
    if (MAPS) {
      store_vec(p.seg_a + (int64_t)seg * p.channels + at.n, va);
      store_vec(p.seg_b + (int64_t)seg * p.channels + at.n, vb);
    } else if (seg == 0 && p.d_c0) {
      store_vec(p.d_c0 + at.n, vb);
    }
  }
}

template <typename T, int VEC, bool GATED>
hipError_t launch_forward(const ScanArgs<T>& p, hipStream_t s) {
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
