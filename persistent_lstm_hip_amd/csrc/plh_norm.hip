// plh_norm.hip -- layer norm over the last dimension, forward and backward.
//
//   xh = (x - mean) rstd        y = xh w + b
//   v = dy w       dx = rstd (v - mean(v) - xh mean(v xh))       dw = sum over rows of dy xh       db = sum of dy
//
// mean and rstd = 1 / sqrt(var + eps) are per row, the variance from the centred values (a second sum over what is in
// registers, so that a large mean costs no digits).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "plh_ops.h"

namespace plh {
namespace {

struct NormArgs {
  const void* x;
  int64_t stride, rows;
  int cols;
  const void *weight, *bias;
  bool w32;  // weight, bias and their gradients are fp32, else of x's type
  float eps, inv_cols;
  void* y;
  float *mean, *rstd;
  const void* d_y;
  void *d_x, *d_weight, *d_bias;
  float* part;  // [groups][2][cols]: the workgroups' sums of dw and db
  int groups;
};

// Sum over the LPR threads of a row, to all of them.  Two sums in turn on two LDS buffers need no barrier of their own
// between rows: every read of one buffer comes before the barrier of the other one's sum.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  constexpr int W = LPR < kWave ? LPR : kWave;
#pragma unroll
  for (int d = 1; d < W; d *= 2) v += __shfl_xor(v, d);
  if constexpr (LPR > kWave) {
    constexpr int N = LPR / kWave;
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    lds_barrier();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) v += lds[i];
  }
  return v;
}

// Two sums of a row at once, with one barrier; the buffers are taken in turn, as above.  (A row's two barriers cost the
// backward pass of 16384 x 8192 bf16 14 us of 166, and 4000 x 12000 fp32, whose workgroup fills a CU, 50 of 171.)
template <int LPR>
__device__ __forceinline__ void row_sums(float& u, float& v, float (*lds)[2]) {
  constexpr int W = LPR < kWave ? LPR : kWave;
#pragma unroll
  for (int d = 1; d < W; d *= 2) {
    u += __shfl_xor(u, d);
    v += __shfl_xor(v, d);
  }
  if constexpr (LPR > kWave) {
    constexpr int N = LPR / kWave;
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave][0] = u, lds[threadIdx.x / kWave][1] = v;
    lds_barrier();
    u = v = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) u += lds[i][0], v += lds[i][1];
  }
}

// sum / cols, corrected by its remainder: the mean of equal values is that value.
__device__ __forceinline__ float mean_of(float sum, const NormArgs& p) {
  const float m = sum * p.inv_cols;
  return fmaf(fmaf(-m, (float)p.cols, sum), p.inv_cols, m);
}

// A parameter vector's VEC elements from column c on.
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, bool p32, int c, float fill, float (&v)[VEC]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = fill;
  } else if (p32) {
    const Vec<float, VEC> t = load_vec<float, VEC>(static_cast<const float*>(p) + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = t.v[j];
  } else {
    const Vec<T, VEC> t = load_vec<T, VEC>(static_cast<const T*>(p) + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)t.v[j];
  }
}

// LPR threads per row, each with NV pieces of VEC neighbouring columns: piece i of thread l is number i LPR + l.  The
// last piece of a row is moved back to end with it; its first `skip` elements then belong to the piece before: they
// are computed and stored by both, and counted once.
template <int VEC, int LPR, int NV>
struct Pieces {
  int col[NV];  // first column; -1: none
  int skip;     // of the thread's last piece

  __device__ __forceinline__ explicit Pieces(int cols) {
    skip = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + (int)threadIdx.x % LPR) * VEC;
      col[i] = c < cols ? min(c, cols - VEC) : -1;
      if (c < cols) skip = c - col[i];
    }
  }
  // Whether element j of piece i counts.  (Only a thread's last piece can be the row's.)
  __device__ __forceinline__ bool counts(int i, int j) const {
    return j >= skip || (i + 1 < NV && col[i + 1] >= 0);
  }
};

template <int LPR>
constexpr int kNormThreads = LPR > 256 ? LPR : 256;

// A workgroup takes rows until none is left, keeps weight and bias in registers, and loads its next row while it
// reduces the one before.  TAIL: VEC does not divide the row length.
template <typename T, int VEC, int LPR, int NV, bool TAIL>
__global__ void __launch_bounds__(kNormThreads<LPR>) norm_forward_kernel(NormArgs p) {
  constexpr int kThreads = kNormThreads<LPR>, kRows = kThreads / LPR;
  __shared__ float lds[2][kThreads / kWave];
  const Pieces<VEC, LPR, NV> at(p.cols);
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (at.col[i] >= 0) {
      load_param<T, VEC>(p.weight, p.w32, at.col[i], 1.0f, w[i]);
      load_param<T, VEC>(p.bias, p.w32, at.col[i], 0.0f, b[i]);
    }
  }
  Vec<T, VEC> next[NV] = {};
  const auto load = [&](int64_t r) __attribute__((always_inline)) {
    if (r >= p.rows) return;
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at.col[i] >= 0) next[i] = load_vec<T, VEC>(src + at.col[i]);
  };
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / LPR;
  const int64_t step = (int64_t)gridDim.x * kRows, rounds = (p.rows + step - 1) / step;
  load(r);
  for (int64_t k = 0; k < rounds; ++k, r += step) {
    float x[NV][VEC], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        x[i][j] = at.col[i] >= 0 ? (float)next[i].v[j] : 0.0f;
        sum += !TAIL || at.counts(i, j) ? x[i][j] : 0.0f;
      }
    }
    if (k + 1 < rounds) load(r + step);
    const float mean = mean_of(row_sum<LPR>(sum, lds[0]), p);
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (at.col[i] >= 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          x[i][j] -= mean;
          if (!TAIL || at.counts(i, j)) sq = fmaf(x[i][j], x[i][j], sq);
        }
      }
    }
    const float rstd = 1.0f / __builtin_sqrtf(fmaf(row_sum<LPR>(sq, lds[1]), p.inv_cols, p.eps));
    if (r >= p.rows) continue;  // (kRows > 1 only: no barrier is skipped)
    T* const dst = static_cast<T*>(p.y) + r * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (at.col[i] >= 0) {
        float y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = fmaf(x[i][j] * rstd, w[i][j], b[i][j]);
        store_vec(dst + at.col[i], round_to<T, VEC>(y));
      }
    }
    if (threadIdx.x % LPR == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}

// Backward.  A row is held as it was loaded and converted again for its second use: that keeps the 16-bit kernels, with
// the next row in flight, at 128 registers and so four waves per SIMD.  32-bit elements take more, and where a
// workgroup's registers run out (1024 threads; 512 with 16 32-bit elements each) the next row is not loaded ahead.  (The
// variant for 513 to 1024 32-bit columns that 4 does not divide spills two registers: 60000 x 1001 takes 147 us, 60000 x
// 1000, whose variant does not, 144.)
template <typename T, int VEC, int LPR, int NV, bool TAIL>
__global__ void __launch_bounds__(kNormThreads<LPR>, sizeof(T) == 2 || LPR == 1024 ? 4 : 3)
    norm_backward_kernel(NormArgs p) {
  constexpr int kThreads = kNormThreads<LPR>, kRows = kThreads / LPR;
  constexpr bool kAhead = LPR < (VEC * NV * sizeof(T) > 32 ? 512 : 1024);
  __shared__ alignas(8) float lds[2][kThreads / kWave][2];
  const Pieces<VEC, LPR, NV> at(p.cols);
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (at.col[i] >= 0) load_param<T, VEC>(p.weight, p.w32, at.col[i], 1.0f, w[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.0f;
  }
  struct Row {
    Vec<T, VEC> x[NV], g[NV];
    float mean, rstd;
  } row = {}, next = {};
  const auto load = [&](Row& to, int64_t r) __attribute__((always_inline)) {
    if (r >= p.rows) return;
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
    const T* const grad = static_cast<const T*>(p.d_y) + r * p.cols;
    to.mean = p.mean[r], to.rstd = p.rstd[r];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (at.col[i] >= 0) {
        to.x[i] = load_vec<T, VEC>(src + at.col[i]);
        to.g[i] = load_vec<T, VEC>(grad + at.col[i]);
      }
    }
  };
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / LPR;
  const int64_t step = (int64_t)gridDim.x * kRows, rounds = (p.rows + step - 1) / step;
  if (kAhead) load(next, r);
  for (int64_t k = 0; k < rounds; ++k, r += step) {
    const bool on = r < p.rows;
    if (kAhead) {
      row = next;
      if (k + 1 < rounds) load(next, r + step);
    } else {
      load(row, r);
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (on && at.col[i] >= 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float g = (float)row.g[i].v[j], xh = ((float)row.x[i].v[j] - row.mean) * row.rstd, v = g * w[i][j];
          dw[i][j] = fmaf(g, xh, dw[i][j]);
          db[i][j] += g;
          if (!TAIL || at.counts(i, j)) {
            s1 += v;
            s2 = fmaf(v, xh, s2);
          }
        }
      }
    }
    row_sums<LPR>(s1, s2, lds[k & 1]);
    const float m1 = s1 * p.inv_cols, m2 = s2 * p.inv_cols;
    if (!on || !p.d_x) continue;
    T* const dst = static_cast<T*>(p.d_x) + r * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (at.col[i] >= 0) {
        float d[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xh = ((float)row.x[i].v[j] - row.mean) * row.rstd;
          d[j] = row.rstd * ((float)row.g[i].v[j] * w[i][j] - m1 - xh * m2);
        }
        store_vec(dst + at.col[i], round_to<T, VEC>(d));
      }
    }
  }
  if (!p.part) return;
  // The rows of a workgroup that ran side by side are summed in their order, then written as one row of partial sums.
  __shared__ float sums[kRows > 1 ? kThreads * VEC * NV : 1];
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float* const out = p.part + (int64_t)blockIdx.x * 2 * p.cols;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if constexpr (kRows > 1) {
      lds_barrier();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[(sub * NV * VEC + i * VEC + j) * LPR + l] = k ? db[i][j] : dw[i][j];
      lds_barrier();
    }
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (at.col[i] >= 0) {
          Vec<float, VEC> t;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float s = k ? db[i][j] : dw[i][j];
            if constexpr (kRows > 1)
              for (int q = 1; q < kRows; ++q) s += sums[(q * NV * VEC + i * VEC + j) * LPR + l];
            t.v[j] = s;
          }
          store_vec(out + (int64_t)k * p.cols + at.col[i], t);
        }
      }
    }
  }
}

// Rows too long for registers: a workgroup per row, which reads it once per sum (again from its XCD's L2: 2000 rows of
// 40000 bf16).
constexpr int kWideThreads = 1024;

// f(vector of N elements' first column) over the thread's columns of a row, whole vectors first.
template <int VEC, typename F>
__device__ __forceinline__ void over_row(int cols, F&& f) {
  const int whole = cols / VEC * VEC;
  for (int c = threadIdx.x * VEC; c < whole; c += kWideThreads * VEC) f(c, std::integral_constant<int, VEC>());
  if (whole + (int)threadIdx.x < cols) f(whole + (int)threadIdx.x, std::integral_constant<int, 1>());
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(NormArgs p) {
  __shared__ float lds[2][kWideThreads / kWave];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
    float s = 0.0f;
    over_row<VEC>(p.cols, [&](int c, auto n) {
      constexpr int N = decltype(n)::value;
      const Vec<T, N> x = load_vec<T, N>(src + c);
#pragma unroll
      for (int j = 0; j < N; ++j) s += (float)x.v[j];
    });
    const float mean = mean_of(row_sum<kWideThreads>(s, lds[0]), p);
    s = 0.0f;
    over_row<VEC>(p.cols, [&](int c, auto n) {
      constexpr int N = decltype(n)::value;
      const Vec<T, N> x = load_vec<T, N>(src + c);
#pragma unroll
      for (int j = 0; j < N; ++j) s = fmaf((float)x.v[j] - mean, (float)x.v[j] - mean, s);
    });
    const float rstd = 1.0f / __builtin_sqrtf(fmaf(row_sum<kWideThreads>(s, lds[1]), p.inv_cols, p.eps));
    over_row<VEC>(p.cols, [&](int c, auto n) {
      constexpr int N = decltype(n)::value;
      const Vec<T, N> x = load_vec<T, N>(src + c);
      float w[N], b[N], y[N];
      load_param<T, N>(p.weight, p.w32, c, 1.0f, w);
      load_param<T, N>(p.bias, p.w32, c, 0.0f, b);
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = fmaf(((float)x.v[j] - mean) * rstd, w[j], b[j]);
      store_vec(static_cast<T*>(p.y) + r * p.cols + c, round_to<T, N>(y));
    });
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kWideThreads) norm_backward_wide_kernel(NormArgs p) {
  __shared__ float lds[2][kWideThreads / kWave];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
    const T* const grad = static_cast<const T*>(p.d_y) + r * p.cols;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    over_row<VEC>(p.cols, [&](int c, auto n) {
      constexpr int N = decltype(n)::value;
      const Vec<T, N> x = load_vec<T, N>(src + c), g = load_vec<T, N>(grad + c);
      float w[N];
      load_param<T, N>(p.weight, p.w32, c, 1.0f, w);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float v = (float)g.v[j] * w[j];
        s1 += v;
        s2 = fmaf(v, ((float)x.v[j] - mean) * rstd, s2);
      }
    });
    const float m1 = row_sum<kWideThreads>(s1, lds[0]) * p.inv_cols;
    const float m2 = row_sum<kWideThreads>(s2, lds[1]) * p.inv_cols;
    over_row<VEC>(p.cols, [&](int c, auto n) {
      constexpr int N = decltype(n)::value;
      const Vec<T, N> x = load_vec<T, N>(src + c), g = load_vec<T, N>(grad + c);
      float w[N], d[N];
      load_param<T, N>(p.weight, p.w32, c, 1.0f, w);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float xh = ((float)x.v[j] - mean) * rstd;
        d[j] = rstd * ((float)g.v[j] * w[j] - m1 - xh * m2);
      }
      store_vec(static_cast<T*>(p.d_x) + r * p.cols + c, round_to<T, N>(d));
    });
  }
}

// The workgroups' sums for such rows: VEC columns per thread (the last thread's moved back to end with the row, as
// above), the rows in as many runs as there are groups.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) norm_columns_kernel(NormArgs p) {
  int c = (blockIdx.x * 256 + threadIdx.x) * VEC;
  if (c >= p.cols) return;
  c = min(c, p.cols - VEC);
  const int64_t per = (p.rows + p.groups - 1) / p.groups;
  const int64_t end = min(p.rows, (blockIdx.y + 1) * per);
  Vec<float, VEC> dw = {}, db = {};
#pragma unroll 2
  for (int64_t r = blockIdx.y * per; r < end; ++r) {
    const Vec<T, VEC> x = load_vec<T, VEC>(static_cast<const T*>(p.x) + r * p.stride + c);
    const Vec<T, VEC> g = load_vec<T, VEC>(static_cast<const T*>(p.d_y) + r * p.cols + c);
    const float mean = p.mean[r], rstd = p.rstd[r];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      dw.v[j] = fmaf((float)g.v[j], ((float)x.v[j] - mean) * rstd, dw.v[j]);
      db.v[j] += (float)g.v[j];
    }
  }
  float* const out = p.part + (int64_t)blockIdx.y * 2 * p.cols;
  store_vec(out + c, dw);
  store_vec(out + p.cols + c, db);
}

// Sums over the workgroups, in a fixed order: 32 threads per column.
template <typename T>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(NormArgs p) {
  __shared__ float lds[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x % 32, n = 2 * (int64_t)p.cols;
  const int q = threadIdx.x / 32;
  float s = 0.0f;
  if (c < n) {
#pragma unroll 8
    for (int g = q; g < p.groups; g += 32) s += p.part[g * n + c];
  }
  lds[q][threadIdx.x % 32] = s;
  lds_barrier();
  if (q != 0 || c >= n) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += lds[i][threadIdx.x];
  void* const dst = c < p.cols ? p.d_weight : p.d_bias;
  const int64_t k = c < p.cols ? c : c - p.cols;
  if (!dst) return;
  if (p.w32)
    static_cast<float*>(dst)[k] = s;
  else
    static_cast<T*>(dst)[k] = round_to<T>(s);
}

// Elements of a piece: 16 bytes, or one element of rows that are shorter than that.
template <typename T>
constexpr int kNormVec = 16 / (int)sizeof(T);

// Threads per row and pieces per thread for `pieces` pieces of VEC columns, up to 16 elements (VEC 8: 2, VEC 4: 4 pieces)
// per thread; {0, 0}: too many for the registers of a workgroup.
struct Shape {
  int lpr, nv;
};
Shape shape_for(int64_t pieces, int vec) {
  for (int lpr : {8, 16, 32, 64})
    if (pieces <= lpr) return {lpr, 1};
  if (pieces <= 128) return {64, 2};
  if (vec == 8) {
    for (int lpr : {256, 512, 1024})
      if (pieces <= 2 * lpr) return {lpr, pieces <= lpr ? 1 : 2};
  } else {
    if (pieces <= 256) return {64, 4};
    for (int lpr : {256, 512, 1024})
      if (pieces <= 4 * lpr) return {lpr, pieces <= 2 * lpr ? 2 : 4};
  }
  return {0, 0};
}

template <typename T, bool BACKWARD, int VEC, int LPR, int NV, bool TAIL>
hipError_t launch_tail(NormArgs p, hipStream_t s) {
  constexpr int kThreads = kNormThreads<LPR>, kRows = kThreads / LPR;
  const int64_t need = (p.rows + kRows - 1) / kRows;
  const unsigned grid = (unsigned)std::min<int64_t>(need, BACKWARD ? p.groups : 256 * (2048 / kThreads));
  if constexpr (BACKWARD)
    hipLaunchKernelGGL((norm_backward_kernel<T, VEC, LPR, NV, TAIL>), dim3(grid), dim3(kThreads), 0, s, p);
  else
    hipLaunchKernelGGL((norm_forward_kernel<T, VEC, LPR, NV, TAIL>), dim3(grid), dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

template <typename T, bool BACKWARD, int VEC>
hipError_t launch_vec(const NormArgs& p, const Shape& sh, hipStream_t s) {
#define PLH_NORM_SHAPE(L, N)                                                 \
  if (sh.lpr == L && sh.nv == N)                                             \
  return p.cols % VEC ? launch_tail<T, BACKWARD, VEC, L, N, true>(p, s) : launch_tail<T, BACKWARD, VEC, L, N, false>(p, s)
  PLH_NORM_SHAPE(8, 1);
  if constexpr (VEC > 1) {
    PLH_NORM_SHAPE(16, 1);
    PLH_NORM_SHAPE(32, 1);
    PLH_NORM_SHAPE(64, 1);
    PLH_NORM_SHAPE(64, 2);
    PLH_NORM_SHAPE(256, 2);
    PLH_NORM_SHAPE(512, 2);
    PLH_NORM_SHAPE(1024, 2);
  }
  if constexpr (VEC == 8) {
    PLH_NORM_SHAPE(256, 1);
  } else if constexpr (VEC == 4) {
    PLH_NORM_SHAPE(64, 4);
    PLH_NORM_SHAPE(256, 4);
    PLH_NORM_SHAPE(512, 4);
    PLH_NORM_SHAPE(1024, 4);
  }
#undef PLH_NORM_SHAPE
  return hipErrorInvalidValue;
}

// Workgroups of the backward pass, of `threads` threads with `side` rows side by side, each with a row of partial sums:
// 1024 threads per CU with one piece per thread, 512 with more (longer rows, whose partial sums weigh more), one
// workgroup at least.  With 512 and 1024 threads per CU: 512000 x 128 fp16 83 and 79 us, 300000 x 129 84 and 68,
// 65536 x 1024 bf16 77 and 82, 7301 x 1001 fp16 16.6 and 18.5, 30000 x 2048 fp32 137 and 145, 16384 x 8192 bf16 153 and
// 163.
int64_t groups_for(int64_t rows, int threads, int side, int nv) {
  const int64_t most = std::max(256, 256 * (nv == 1 ? 1024 : 512) / threads);
  return std::max<int64_t>(1, std::min<int64_t>((rows + side - 1) / side, most));
}
constexpr int kWideGroups = 64;  // runs of rows of norm_columns_kernel

// How a call with pieces of `v` columns (16 bytes) is laid out.
struct NormLayout {
  int vec;      // columns of a piece: v, or one where a row is shorter than that
  Shape shape;  // {0, 0}: a workgroup per row
  int groups;   // rows of partial sums of the backward pass, one at least
};
NormLayout norm_layout(int v, int64_t rows, int64_t cols) {
  NormLayout l;
  l.vec = cols >= v ? v : 1;
  l.shape = shape_for((cols + l.vec - 1) / l.vec, l.vec);
  const int threads = std::max(l.shape.lpr, 256);
  l.groups = l.shape.lpr ? (int)groups_for(rows, threads, threads / l.shape.lpr, l.shape.nv)
                         : (int)std::max<int64_t>(1, std::min<int64_t>(rows, kWideGroups));
  return l;
}

template <typename T, bool BACKWARD>
hipError_t launch_norm(NormArgs p, hipStream_t s) {
  constexpr int V = kNormVec<T>;
  const NormLayout l = norm_layout(V, p.rows, p.cols);
  p.groups = l.groups;
  if (BACKWARD && !p.d_weight && !p.d_bias) p.part = nullptr;
  hipError_t e = hipSuccess;
  if (l.shape.lpr) {
    e = l.vec == V ? launch_vec<T, BACKWARD, V>(p, l.shape, s) : launch_vec<T, BACKWARD, 1>(p, l.shape, s);
  } else {
    const unsigned grid = (unsigned)std::min<int64_t>(p.rows, 1024);
    if constexpr (!BACKWARD) {
      hipLaunchKernelGGL((norm_forward_wide_kernel<T, V>), dim3(grid), dim3(kWideThreads), 0, s, p);
      e = hipGetLastError();
    } else {
      if (p.d_x) {
        hipLaunchKernelGGL((norm_backward_wide_kernel<T, V>), dim3(grid), dim3(kWideThreads), 0, s, p);
        e = hipGetLastError();
      }
      if (e == hipSuccess && p.part) {
        hipLaunchKernelGGL((norm_columns_kernel<T, V>), dim3((p.cols + 256 * V - 1) / (256 * V), p.groups), dim3(256), 0,
                           s, p);
        e = hipGetLastError();
      }
    }
  }
  if (e == hipSuccess && BACKWARD && p.part) {
    hipLaunchKernelGGL(norm_reduce_kernel<T>, dim3((unsigned)((2 * (int64_t)p.cols + 31) / 32)), dim3(1024), 0, s, p);
    e = hipGetLastError();
  }
  return e;
}

int check_norm(const char* what, int dtype, int wdtype, int64_t stride, int64_t rows, int64_t cols,
               const void* x) noexcept {
  if (dtype != PLH_F16 && dtype != PLH_BF16 && dtype != PLH_F32)
    return op_error(PLH_ERR_INVALID, what, "dtype must be PLH_F16, PLH_BF16 or PLH_F32");
  if (wdtype != dtype && wdtype != PLH_F32) return op_error(PLH_ERR_INVALID, what, "wdtype must be dtype or PLH_F32");
  if (rows < 0) return op_error(PLH_ERR_INVALID, what, "rows must be non-negative");
  if (cols < 1 || cols > (1 << 24)) return op_error(PLH_ERR_UNSUPPORTED, what, "cols must lie in [1, 2^24]");
  if (rows > 0 && !x) return op_error(PLH_ERR_INVALID, what, "x is required");
  if (stride < 0) return op_error(PLH_ERR_INVALID, what, "stride must be non-negative");
  return PLH_OK;
}

}  // namespace
}  // namespace plh

extern "C" {

int64_t plh_layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1 || cols > (1 << 24)) return -1;
  int groups = 0;  // the most of any type
  for (int v : {plh::kNormVec<_Float16>, plh::kNormVec<float>})
    groups = std::max(groups, plh::norm_layout(v, rows, cols).groups);
  return groups * 2 * cols * (int64_t)sizeof(float);
}

int plh_layer_norm_forward(int dtype, int wdtype, const void* x, int64_t stride, int64_t rows, int64_t cols,
                           const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd,
                           void* stream) {
  const char* const what = "layer_norm_forward";
  const int rc = plh::check_norm(what, dtype, wdtype, stride, rows, cols, x);
  if (rc != PLH_OK) return rc;
  if (rows == 0) return PLH_OK;
  if (!y) return plh::op_error(PLH_ERR_INVALID, what, "y is required");
  plh::NormArgs p = {};
  p.x = x, p.stride = stride, p.rows = rows, p.cols = (int)cols;
  p.weight = weight, p.bias = bias, p.w32 = wdtype == PLH_F32;
  p.eps = eps, p.inv_cols = 1.0f / (float)cols;
  p.y = y, p.mean = mean, p.rstd = rstd;
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) { e = plh::launch_norm<decltype(zero), false>(p, (hipStream_t)stream); });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

int plh_layer_norm_backward(int dtype, int wdtype, const void* x, int64_t stride, int64_t rows, int64_t cols,
                            const void* weight, const float* mean, const float* rstd, const void* d_y, void* d_x,
                            void* d_weight, void* d_bias, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* const what = "layer_norm_backward";
  const int rc = plh::check_norm(what, dtype, wdtype, stride, rows, cols, x);
  if (rc != PLH_OK) return rc;
  if (rows > 0 && (!mean || !rstd || !d_y))
    return plh::op_error(PLH_ERR_INVALID, what, "mean, rstd and d_y are required");
  if ((d_weight || d_bias) && (!workspace || workspace_bytes < plh_layer_norm_workspace_bytes(rows, cols)))
    return plh::op_error(PLH_ERR_INVALID, what, "workspace missing or smaller than plh_layer_norm_workspace_bytes()");
  if (!plh::aligned(workspace, 16))
    return plh::op_error(PLH_ERR_INVALID, what, "workspace must be 16-byte aligned");
  plh::NormArgs p = {};
  p.x = x, p.stride = stride, p.rows = rows, p.cols = (int)cols;
  p.weight = weight, p.w32 = wdtype == PLH_F32, p.inv_cols = 1.0f / (float)cols;
  p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd);
  p.d_y = d_y, p.d_x = d_x, p.d_weight = d_weight, p.d_bias = d_bias, p.part = (float*)workspace;
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (rows > 0) {
      e = plh::launch_norm<T, true>(p, (hipStream_t)stream);
    } else if (d_weight || d_bias) {  // no rows: the sums are zero (groups = 0)
      hipLaunchKernelGGL(plh::norm_reduce_kernel<T>, dim3((unsigned)((2 * cols + 31) / 32)), dim3(1024), 0,
                         (hipStream_t)stream, p);
      e = hipGetLastError();
    }
  });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}

}  // extern "C"
