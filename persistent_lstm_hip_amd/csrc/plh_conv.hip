// plh_conv.hip -- short causal convolution along time, a filter of 1 to 8 taps per channel, forward, backward and for
// one token.
//
//   acc_t = bias + sum_k w_k x_{t-W+1+k}      y_t = silu(acc_t) = acc_t sigmoid(acc_t)   (or y_t = acc_t)
//
// x before the first step comes from a state, the W - 1 inputs before it (zeros without one); the new state is the last
// W - 1 inputs of the row.  Gradients, with da_t = dy_t silu'(acc_t), zero outside the row:
//   dx_t = sum_k w_k da_{t+W-1-k}      dw_k = sum_t da_t x_{t-W+1+k}      db = sum_t da_t
// and the new state's gradient is added to the inputs that it holds.  acc is computed again where the gradient needs
// it (W products for two bytes less to write and to read).
//
// Everything is bound by the memory traffic: x in, y out (dy in and dx out).  A thread has four neighbouring channels and
// walks along time with the last W - 1 inputs in registers, so that an input is read once but for the W - 1 at the edges of
// its stretch.  512 rows of 1000 steps x 256 channels fp16, W = 4: forward 103 us (5.1 TB/s), backward 184 (4.3); with rows
// of 200 to 1000 steps 87 and 179.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "plh_ops.h"

namespace plh {
namespace {

constexpr int kMaxWidth = 8;
constexpr int kStep = 4;  // steps that a thread loads at once

struct ConvArgs {
  const void* x;
  int64_t stride_b, stride_t;  // elements
  int64_t batch;
  int T_, C, pieces;
  const void *weight, *bias;
  bool w32, silu;
  const void* state;  // [B][W - 1][C] or null
  const int32_t* lengths;
  void *y, *state_n;
  int stretch, stretches;  // steps of a thread (a multiple of kStep), stretches of a row
  uint32_t blocks;         // that compute y; the ones after them write state_n
  const void *d_y, *d_state_n;  // backward
  void *d_x, *d_state;
  float* part;  // [groups][C W + C]: the workgroups' sums of dw and db
  int groups, units;  // workgroups that share a slab of channels; stretches of all rows
  void *d_weight, *d_bias;
};

__device__ __forceinline__ int row_length(const ConvArgs& p, int64_t b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.T_) : p.T_;
}

// The filters of VEC channels, [channel][tap] in memory.
template <typename T, int VEC, int W>
__device__ __forceinline__ void load_filters(const ConvArgs& p, int c, float (&w)[W][VEC]) {
  const auto load = [&](auto zero) __attribute__((always_inline)) {
    using F = decltype(zero);
    const Vec<F, VEC * W> v = load_vec<F, VEC * W>(static_cast<const F*>(p.weight) + (int64_t)c * W);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
#pragma unroll
      for (int k = 0; k < W; ++k) w[k][j] = (float)v.v[j * W + k];
  };
  if (p.w32)
    load(float());
  else
    load(T());
}

template <typename T, int VEC>
__device__ __forceinline__ void to_float(const Vec<T, VEC>& v, float (&f)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = (float)v.v[j];
}

// The input at position t of row b (negative: in the state), zero outside the row [-(W - 1), len).
template <typename T, int VEC, int W>
__device__ __forceinline__ Vec<T, VEC> load_input(const ConvArgs& p, int64_t b, int t, int len, int c) {
  Vec<T, VEC> v = {};
  if (t >= 0) {
    if (t < len) v = load_vec<T, VEC>(static_cast<const T*>(p.x) + b * p.stride_b + (int64_t)t * p.stride_t + c);
  } else if (W > 1 && p.state) {
    v = load_vec<T, VEC>(static_cast<const T*>(p.state) + (b * (W - 1) + t + W - 1) * p.C + c);
  }
  return v;
}

// kStep steps from step t on, of a row of len steps; src moves on.  (One check for all of them, and a pointer that moves:
// every step's own take more instructions than the filter, backward 246 -> 229 us at the sizes above, ragged.)
template <typename T, int VEC>
__device__ __forceinline__ void load_steps(const T*& src, int64_t stride, int t, int len, Vec<T, VEC> (&v)[kStep]) {
  if (t + kStep <= len) {
#pragma unroll
    for (int s = 0; s < kStep; ++s) v[s] = load_vec<T, VEC>(src + s * stride);
  } else {
#pragma unroll
    for (int s = 0; s < kStep; ++s) {
      v[s] = Vec<T, VEC>{};
      if (t + s < len) v[s] = load_vec<T, VEC>(src + s * stride);
    }
  }
  src += kStep * stride;
}

// ---- forward ------------------------------------------------------------------------------------

template <typename T, int VEC, int W, bool SILU>
__global__ void __launch_bounds__(256) conv_forward_kernel(ConvArgs p) {
  const uint32_t block = blockIdx.x;
  if (W > 1 && block >= p.blocks) {  // the new state: a piece per thread
    const int64_t i = (int64_t)(block - p.blocks) * 256 + threadIdx.x, rest = i / p.pieces;
    if (rest >= p.batch * (W - 1)) return;
    const int c = min((int)(i % p.pieces) * VEC, p.C - VEC), j = (int)(rest % max(W - 1, 1));
    const int64_t b = rest / max(W - 1, 1);
    const int len = row_length(p, b);
    store_vec(static_cast<T*>(p.state_n) + rest * p.C + c, load_input<T, VEC, W>(p, b, len - (W - 1) + j, len, c));
    return;
  }
  const uint32_t i = block * 256 + threadIdx.x, unit = i / (uint32_t)p.pieces;  // (less than 2^32 of them)
  const int64_t b = unit / (uint32_t)p.stretches;
  if (b >= p.batch) return;
  const int c = min((int)(i % (uint32_t)p.pieces) * VEC, p.C - VEC);
  const int begin = (int)(unit % (uint32_t)p.stretches) * p.stretch, end = min(begin + p.stretch, p.T_);
  const int len = row_length(p, b);
  T* const y = static_cast<T*>(p.y) + (b * p.T_ + begin) * p.C + c;
  const int live_end = max(begin, min(end, len));
  for (int t = live_end; t < end; ++t) store_vec(y + (int64_t)(t - begin) * p.C, Vec<T, VEC>{});
  if (live_end == begin) return;
  float w[W][VEC], bias[VEC], x[W - 1 + kStep][VEC];
  load_filters<T, VEC, W>(p, c, w);
  load_param<T, VEC>(p.bias, p.w32, c, 0.0f, bias);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) to_float(load_input<T, VEC, W>(p, b, begin - (W - 1) + k, len, c), x[k]);
  Vec<T, VEC> next[kStep];
  const T* src = static_cast<const T*>(p.x) + b * p.stride_b + (int64_t)begin * p.stride_t + c;
  T* dst = y;
  const auto load = [&](int t) __attribute__((always_inline)) { load_steps(src, p.stride_t, t, len, next); };
  const auto steps = [&](auto inside, int t) __attribute__((always_inline)) {
    constexpr bool INSIDE = decltype(inside)::value;  // none of the steps lies past live_end
#pragma unroll
    for (int s = 0; s < kStep; ++s) {
      if (!INSIDE && t + s >= live_end) continue;
      float out[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float acc = bias[j];
#pragma unroll
        for (int k = 0; k < W; ++k) acc = fmaf(w[k][j], x[s + k][j], acc);
        out[j] = SILU ? silu(acc) : acc;
      }
      store_vec(dst + (int64_t)s * p.C, round_to<T, VEC>(out));
    }
    dst += (int64_t)kStep * p.C;
  };
  load(begin);
  for (int t = begin; t < live_end; t += kStep) {
#pragma unroll
    for (int s = 0; s < kStep; ++s) to_float(next[s], x[W - 1 + s]);
    if (t + kStep < live_end) load(t + kStep);
    if (t + kStep <= live_end)
      steps(std::true_type(), t);
    else
      steps(std::false_type(), t);
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[k][j] = x[k + kStep][j];
  }
}

// ---- one token ----------------------------------------------------------------------------------

// A thread per piece of a row; a row's last piece may be shorter (it is not moved back: two threads would then update
// the same channels of a state in place).
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(256) conv_step_kernel(ConvArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, b = i / p.pieces;
  if (b >= p.batch) return;
  const int first = (int)(i % p.pieces) * VEC;
  const auto run = [&](int c, auto n) __attribute__((always_inline)) {
    constexpr int N = decltype(n)::value;
    float w[W][N], acc[N], v[N];
    Vec<T, N> x[W];
    const T* const state = static_cast<const T*>(p.state) + b * (W - 1) * p.C + c;
    T* const state_n = static_cast<T*>(p.state_n) + b * (W - 1) * p.C + c;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) x[k] = load_vec<T, N>(state + (int64_t)k * p.C);
    x[W - 1] = load_vec<T, N>(static_cast<const T*>(p.x) + b * p.stride_b + c);
    load_filters<T, N, W>(p, c, w);
    load_param<T, N>(p.bias, p.w32, c, 0.0f, acc);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      to_float(x[k], v);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = fmaf(w[k][j], v[j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = p.silu ? silu(acc[j]) : acc[j];
    store_vec(static_cast<T*>(p.y) + b * p.C + c, round_to<T, N>(acc));
#pragma unroll
    for (int k = 0; k < W - 1; ++k) store_vec(state_n + (int64_t)k * p.C, x[k + 1]);
  };
  if (first + VEC <= p.C)
    run(first, std::integral_constant<int, VEC>());
  else
    for (int c = first; c < p.C; ++c) run(c, std::integral_constant<int, 1>());
}

// ---- backward -----------------------------------------------------------------------------------

// Threads of a workgroup side by side in the channels (a slab), and stretches that it works on at once.
struct ConvGroup {
  int ct, tg;
};

// A workgroup has a slab of CT pieces of channels and, TG at a time, the stretches of all rows that its number gives
// it; it keeps its sums of dw and db in registers until the end.
template <typename T, int VEC, int W, int CT, bool SILU>
__global__ void __launch_bounds__(256) conv_backward_kernel(ConvArgs p) {
  constexpr int TG = 256 / CT;
  const int slabs = (p.pieces + CT - 1) / CT, slab = blockIdx.x % slabs, group = blockIdx.x / slabs;
  const int ct = threadIdx.x % CT, tg = threadIdx.x / CT, piece = slab * CT + ct;
  const bool on = piece < p.pieces;
  const int c = on ? min(piece * VEC, p.C - VEC) : 0;
  float w[W][VEC], bias[VEC], dw[W][VEC], db[VEC];
  load_filters<T, VEC, W>(p, c, w);
  load_param<T, VEC>(p.bias, p.w32, c, 0.0f, bias);
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    db[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][j] = 0.0f;
  }
  const int step = p.groups * TG;
  for (int unit = group * TG + tg; unit < p.units && on; unit += step) {
    const int64_t b = unit / p.stretches;
    const int begin = unit % p.stretches * p.stretch, end = min(begin + p.stretch, p.T_);
    const int len = row_length(p, b);
    const int64_t at = (b * p.T_ + begin) * p.C + c;
    const T *src = static_cast<const T*>(p.x) + b * p.stride_b + (int64_t)begin * p.stride_t + c,
            *grad = static_cast<const T*>(p.d_y) + at;
    T* d_x = p.d_x ? static_cast<T*>(p.d_x) + at - (int64_t)(W - 1) * p.C : nullptr;  // of position t - (W - 1)
    T* const d_state = W > 1 && p.d_state && begin == 0 ? static_cast<T*>(p.d_state) + b * (W - 1) * p.C + c : nullptr;
    const int live_end = max(begin, min(end, len));
    if (p.d_x)
      for (int t = live_end; t < end; ++t)
        store_vec(static_cast<T*>(p.d_x) + at + (int64_t)(t - begin) * p.C, Vec<T, VEC>{});
    if (live_end == begin && !d_state) continue;
    // Position t of the walk: da_t, whose dx is complete for position t - (W - 1).  A stretch is walked W - 1 positions
    // past its (or the row's) end; the first one gives the state's gradient too.
    float x[W - 1 + kStep][VEC], da[W - 1 + kStep][VEC];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      to_float(load_input<T, VEC, W>(p, b, begin - (W - 1) + k, len, c), x[k]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) da[k][j] = 0.0f;
    }
    Vec<T, VEC> nx[kStep], ng[kStep];
    const auto load = [&](int t) __attribute__((always_inline)) {
      load_steps(src, p.stride_t, t, len, nx);
      load_steps(grad, (int64_t)p.C, t, len, ng);
    };
    const auto steps = [&](auto inside, int t) __attribute__((always_inline)) {
      constexpr bool INSIDE = decltype(inside)::value;  // all of the steps lie in the row and in the stretch, and so do
#pragma unroll                                          // the positions whose dx they complete
      for (int s = 0; s < kStep; ++s) {
        const bool live = INSIDE || t + s < len;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float& g = da[W - 1 + s][j];
          if (SILU) {
            float acc = bias[j];
#pragma unroll
            for (int k = 0; k < W; ++k) acc = fmaf(w[k][j], x[s + k][j], acc);
            g *= silu_slope(acc);
          }
          if (!INSIDE) g = live ? g : 0.0f;
        }
        if (INSIDE || (live && t + s < end)) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            db[j] += da[W - 1 + s][j];
#pragma unroll
            for (int k = 0; k < W; ++k) dw[k][j] = fmaf(da[W - 1 + s][j], x[s + k][j], dw[k][j]);
          }
        }
        const int q = t + s - (W - 1);
        if (!INSIDE && (q >= live_end || (q < begin && !d_state))) continue;
        float out[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          out[j] = w[0][j] * da[s + W - 1][j];
#pragma unroll
          for (int k = 1; k < W; ++k) out[j] = fmaf(w[k][j], da[s + W - 1 - k][j], out[j]);
        }
        if (!INSIDE && W > 1 && p.d_state_n && q >= len - (W - 1)) {
          float extra[VEC];
          to_float(load_vec<T, VEC>(static_cast<const T*>(p.d_state_n) + (b * (W - 1) + q - len + W - 1) * p.C + c), extra);
#pragma unroll
          for (int j = 0; j < VEC; ++j) out[j] += extra[j];
        }
        if (W > 1 && !INSIDE && q < 0)
          store_vec(d_state + (int64_t)(q + W - 1) * p.C, round_to<T, VEC>(out));
        else if (d_x)
          store_vec(d_x + (int64_t)s * p.C, round_to<T, VEC>(out));
      }
      if (d_x) d_x += (int64_t)kStep * p.C;
    };
    const int last = live_end + W - 1;
    load(begin);
    for (int t = begin; t < last; t += kStep) {
#pragma unroll
      for (int s = 0; s < kStep; ++s) {
        to_float(nx[s], x[W - 1 + s]);
        to_float(ng[s], da[W - 1 + s]);
      }
      if (t + kStep < last) load(t + kStep);
      if (t - (W - 1) >= begin && t + kStep <= live_end)
        steps(std::true_type(), t);
      else
        steps(std::false_type(), t);
#pragma unroll
      for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[k][j] = x[k + kStep][j], da[k][j] = da[k + kStep][j];
    }
  }
  if (!p.part) return;
  // The stretches' sums, added in their order.
  __shared__ float lds[(W + 1) * VEC][256];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
#pragma unroll
    for (int k = 0; k < W; ++k) lds[j * W + k][threadIdx.x] = dw[k][j];
    lds[VEC * W + j][threadIdx.x] = db[j];
  }
  lds_barrier();
  float* const out = p.part + (int64_t)group * p.C * (W + 1);
  for (int i = tg; i < (W + 1) * VEC && on; i += TG) {
    float sum = 0.0f;
    for (int q = 0; q < TG; ++q) sum += lds[i][q * CT + ct];
    if (i < W * VEC)
      out[(int64_t)c * W + i] = sum;
    else
      out[(int64_t)p.C * W + c + i - W * VEC] = sum;
  }
}

// ---- host ---------------------------------------------------------------------------------------

// Channels of a thread: wider pieces (16 bytes) take the registers that hide the loads' latency (512 x 1000 x 256 fp16,
// W = 4, ragged, forward 107 us with eight channels, 92 with four, 89 with two; backward 229, 221 and 217).
constexpr int kConvVec = 4, kConvStepVec = 4;

// f(std::integral_constant of the width).
template <typename F>
hipError_t with_width(int width, F&& f) {
  switch (width) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    case 4: return f(std::integral_constant<int, 4>());
    case 5: return f(std::integral_constant<int, 5>());
    case 6: return f(std::integral_constant<int, 6>());
    case 7: return f(std::integral_constant<int, 7>());
    case 8: return f(std::integral_constant<int, 8>());
    default: return hipErrorInvalidValue;
  }
}

// Steps of a thread's stretch: long ones read fewer inputs twice, short ones make more threads, among which rows of unequal
// length are shared more evenly (at the sizes above, ragged, forward with 16, 32 and 64 steps 85, 101 and 107 us, all rows
// full 103, 110 and 117).
int stretch_for(int64_t batch, int64_t seq_len, int64_t pieces, int64_t threads, int most) {
  const int64_t want = batch * pieces * seq_len / std::max<int64_t>(threads, 1);  // steps per thread that fill the device
  const int64_t steps = std::min<int64_t>(std::max<int64_t>(want, kStep), most);
  return (int)((steps + kStep - 1) / kStep * kStep);
}

template <typename T>
hipError_t launch_conv_forward(ConvArgs p, int width, hipStream_t s) {
  const auto run = [&](auto v) {
    constexpr int VEC = decltype(v)::value;
    p.pieces = (p.C + VEC - 1) / VEC;
    p.stretch = stretch_for(p.batch, p.T_, p.pieces, 256 * 1024, 16);
    p.stretches = (p.T_ + p.stretch - 1) / p.stretch;
    p.blocks = (uint32_t)((p.batch * p.stretches * p.pieces + 255) / 256);
    const int64_t state_blocks = (p.batch * (width - 1) * p.pieces + 255) / 256;
    const dim3 grid((unsigned)(p.blocks + state_blocks));
    if (grid.x == 0) return hipSuccess;
    return with_width(width, [&](auto w) {
      if (p.silu)
        hipLaunchKernelGGL((conv_forward_kernel<T, VEC, decltype(w)::value, true>), grid, dim3(256), 0, s, p);
      else
        hipLaunchKernelGGL((conv_forward_kernel<T, VEC, decltype(w)::value, false>), grid, dim3(256), 0, s, p);
      return hipGetLastError();
    });
  };
  return p.C >= kConvVec ? run(std::integral_constant<int, kConvVec>()) : run(std::integral_constant<int, 1>());
}

template <typename T>
hipError_t launch_conv_step(ConvArgs p, int width, hipStream_t s) {
  constexpr int VEC = kConvStepVec;
  p.pieces = (p.C + VEC - 1) / VEC;
  const dim3 grid((unsigned)((p.batch * p.pieces + 255) / 256));
  return with_width(width, [&](auto w) {
    hipLaunchKernelGGL((conv_step_kernel<T, VEC, decltype(w)::value>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
  });
}

// How a backward call is laid out, the same for every type.
struct ConvLayout {
  int vec, pieces, ct, slabs, stretch, stretches, groups;
  int64_t units;
};
ConvLayout conv_layout(int64_t batch, int64_t seq_len, int64_t channels) {
  ConvLayout l;
  l.vec = channels >= kConvVec ? kConvVec : 1;
  l.pieces = (int)((channels + l.vec - 1) / l.vec);
  l.ct = l.pieces > 16 ? 32 : l.pieces > 8 ? 16 : 8;
  l.slabs = (l.pieces + l.ct - 1) / l.ct;
  l.stretch = stretch_for(batch, seq_len, l.pieces, 256 * 1024, 64);
  l.stretches = (int)((seq_len + l.stretch - 1) / l.stretch);
  l.units = batch * l.stretches;
  // (with 1024 and 2048 workgroups the ragged rows above take 193 and 179 us)
  const int64_t tg = 256 / l.ct, most = std::max<int64_t>(1, 2048 / l.slabs);
  l.groups = (int)std::max<int64_t>(1, std::min<int64_t>((l.units + tg - 1) / tg, most));
  return l;
}

template <typename T>
hipError_t launch_conv_backward(ConvArgs p, int width, hipStream_t s) {
  const ConvLayout l = conv_layout(p.batch, p.T_, p.C);
  p.pieces = l.pieces, p.stretch = l.stretch, p.stretches = l.stretches, p.groups = l.groups, p.units = (int)l.units;
  if (!p.d_weight && !p.d_bias) p.part = nullptr;
  const dim3 grid((unsigned)(l.slabs * l.groups));
  hipError_t e = with_width(width, [&](auto w) {
    constexpr int W = decltype(w)::value;
    const auto run = [&](auto v, auto ct) {
      constexpr int VEC = decltype(v)::value, CT = decltype(ct)::value;
      if (p.silu)
        hipLaunchKernelGGL((conv_backward_kernel<T, VEC, W, CT, true>), grid, dim3(256), 0, s, p);
      else
        hipLaunchKernelGGL((conv_backward_kernel<T, VEC, W, CT, false>), grid, dim3(256), 0, s, p);
    };
    const auto vec = [&](auto v) {
      if (l.ct == 32)
        run(v, std::integral_constant<int, 32>());
      else if (l.ct == 16)
        run(v, std::integral_constant<int, 16>());
      else
        run(v, std::integral_constant<int, 8>());
    };
    if (l.vec == kConvVec)
      vec(std::integral_constant<int, kConvVec>());
    else
      run(std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
    return hipGetLastError();
  });
  if (e == hipSuccess && p.part) {
    ColumnSums sums = {};
    sums.part = p.part, sums.rows = p.batch > 0 && p.T_ > 0 ? l.groups : 0;
    sums.cols = (int64_t)p.C * (width + 1), sums.out32 = p.w32;
    sums.out[0] = p.d_weight, sums.begin[1] = (int64_t)p.C * width, sums.out[1] = p.d_bias;
    sums.begin[2] = sums.begin[3] = sums.cols;
    e = launch_column_sums<T>(sums, s);
  }
  return e;
}

int check_conv(const char* what, int dtype, int wdtype, const void* x, int64_t stride_b, int64_t stride_t, int64_t batch,
               int64_t seq_len, int64_t channels, int width, const void* weight) noexcept {
  if (dtype != PLH_F16 && dtype != PLH_BF16 && dtype != PLH_F32)
    return op_error(PLH_ERR_INVALID, what, "dtype must be PLH_F16, PLH_BF16 or PLH_F32");
  if (wdtype != dtype && wdtype != PLH_F32) return op_error(PLH_ERR_INVALID, what, "wdtype must be dtype or PLH_F32");
  if (batch < 0 || seq_len < 0) return op_error(PLH_ERR_INVALID, what, "batch and seq_len must be non-negative");
  if (width < 1 || width > kMaxWidth) return op_error(PLH_ERR_UNSUPPORTED, what, "width must lie in [1, 8]");
  if (channels < 1 || channels > (1 << 22)) return op_error(PLH_ERR_UNSUPPORTED, what, "channels must lie in [1, 2^22]");
  if (seq_len > (1 << 30)) return op_error(PLH_ERR_UNSUPPORTED, what, "seq_len must not exceed 2^30");
  if (batch > (1 << 28) || batch * channels > (1 << 28) ||
      (seq_len > 0 && batch * channels > (int64_t(1) << 35) / seq_len))
    return op_error(PLH_ERR_UNSUPPORTED, what,
                    "batch * channels must not exceed 2^28, batch * channels * seq_len not 2^35");
  if (batch > 0 && seq_len > 0 && !x) return op_error(PLH_ERR_INVALID, what, "x is required");
  if (!weight) return op_error(PLH_ERR_INVALID, what, "weight is required");
  if (stride_b < 0 || stride_t < 0) return op_error(PLH_ERR_INVALID, what, "strides must be non-negative");
  return PLH_OK;
}

ConvArgs conv_args(int wdtype, const void* x, int64_t stride_b, int64_t stride_t, int64_t batch, int64_t seq_len,
                   int64_t channels, const void* weight, const void* bias, const void* state, const int32_t* lengths,
                   int silu) {
  ConvArgs p = {};
  p.x = x, p.stride_b = stride_b, p.stride_t = stride_t, p.batch = batch, p.T_ = (int)seq_len, p.C = (int)channels;
  p.weight = weight, p.bias = bias, p.w32 = wdtype == PLH_F32, p.silu = silu != 0;
  p.state = state, p.lengths = lengths;
  return p;
}

}  // namespace
}  // namespace plh

extern "C" {

int64_t plh_causal_conv_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int width) {
  if (batch < 0 || seq_len < 0 || seq_len > (1 << 30) || channels < 1 || channels > (1 << 22) || width < 1 ||
      width > plh::kMaxWidth)
    return -1;
  return plh::conv_layout(batch, seq_len, channels).groups * channels * (width + 1) * (int64_t)sizeof(float);
}

int plh_causal_conv_forward(int dtype, int wdtype, const void* x, int64_t stride_b, int64_t stride_t, int64_t batch,
                            int64_t seq_len, int64_t channels, int width, const void* weight, const void* bias,
                            const void* state, const int32_t* lengths, int silu, void* y, void* state_n, void* stream) {
  const char* const what = "causal_conv_forward";
  const int rc = plh::check_conv(what, dtype, wdtype, x, stride_b, stride_t, batch, seq_len, channels, width, weight);
  if (rc != PLH_OK) return rc;
  if (batch == 0) return PLH_OK;
  if ((seq_len > 0 && !y) || (width > 1 && !state_n))
    return plh::op_error(PLH_ERR_INVALID, what, "y and state_n are required");
  plh::ConvArgs p = plh::conv_args(wdtype, x, stride_b, stride_t, batch, seq_len, channels, weight, bias, state, lengths,
                                   silu);
  p.y = y, p.state_n = state_n;
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) { e = plh::launch_conv_forward<decltype(zero)>(p, width, (hipStream_t)stream); });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

int plh_causal_conv_step(int dtype, int wdtype, const void* x, int64_t stride_b, int64_t batch, int64_t channels, int width,
                         const void* weight, const void* bias, const void* state, int silu, void* y, void* state_n,
                         void* stream) {
  const char* const what = "causal_conv_step";
  const int rc = plh::check_conv(what, dtype, wdtype, x, stride_b, 0, batch, 1, channels, width, weight);
  if (rc != PLH_OK) return rc;
  if (batch == 0) return PLH_OK;
  if (!y || (width > 1 && (!state || !state_n)))
    return plh::op_error(PLH_ERR_INVALID, what, "state, y and state_n are required");
  plh::ConvArgs p = plh::conv_args(wdtype, x, stride_b, 0, batch, 1, channels, weight, bias, state, nullptr, silu);
  p.y = y, p.state_n = state_n;
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) { e = plh::launch_conv_step<decltype(zero)>(p, width, (hipStream_t)stream); });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

int plh_causal_conv_backward(int dtype, int wdtype, const void* x, int64_t stride_b, int64_t stride_t, int64_t batch,
                             int64_t seq_len, int64_t channels, int width, const void* weight, const void* bias,
                             const void* state, const int32_t* lengths, int silu, const void* d_y, const void* d_state_n,
                             void* d_x, void* d_weight, void* d_bias, void* d_state, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const char* const what = "causal_conv_backward";
  const int rc = plh::check_conv(what, dtype, wdtype, x, stride_b, stride_t, batch, seq_len, channels, width, weight);
  if (rc != PLH_OK) return rc;
  if (batch > 0 && seq_len > 0 && !d_y) return plh::op_error(PLH_ERR_INVALID, what, "d_y is required");
  if (seq_len == 0 && d_state) return plh::op_error(PLH_ERR_UNSUPPORTED, what, "d_state needs at least one step");
  if ((d_weight || d_bias) &&
      (!workspace || workspace_bytes < plh_causal_conv_workspace_bytes(batch, seq_len, channels, width)))
    return plh::op_error(PLH_ERR_INVALID, what, "workspace missing or smaller than plh_causal_conv_workspace_bytes()");
  if (!plh::aligned(workspace, 16)) return plh::op_error(PLH_ERR_INVALID, what, "workspace must be 16-byte aligned");
  plh::ConvArgs p = plh::conv_args(wdtype, x, stride_b, stride_t, batch, seq_len, channels, weight, bias, state, lengths,
                                   silu);
  p.d_y = d_y, p.d_state_n = d_state_n, p.d_x = d_x, p.d_weight = d_weight, p.d_bias = d_bias, p.d_state = d_state;
  p.part = (float*)workspace;
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) { e = plh::launch_conv_backward<decltype(zero)>(p, width, (hipStream_t)stream); });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

}  // extern "C"
