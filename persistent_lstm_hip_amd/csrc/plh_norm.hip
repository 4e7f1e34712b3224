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
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) v += lds[i];
  }
  return v;
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
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = static_cast<const float*>(p)[c + j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)static_cast<const T*>(p)[c + j];
  }
}

// LPR threads per row, each with NV pieces of VEC neighbouring columns: piece i of thread l starts at column
// (i LPR + l) VEC.  A workgroup takes rows until none is left and keeps weight and bias in registers.
template <typename T, int VEC, int LPR, int NV>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256) norm_forward_kernel(NormArgs p) {
  constexpr int kThreads = LPR > 256 ? LPR : 256, kRows = kThreads / LPR;
  __shared__ float lds[2][kThreads / kWave];
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LPR + l) * VEC;
    if (c < p.cols) {
      load_param<T, VEC>(p.weight, p.w32, c, 1.0f, w[i]);
      load_param<T, VEC>(p.bias, p.w32, c, 0.0f, b[i]);
    }
  }
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < p.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t r = base + sub;
    const bool on = r < p.rows;
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
    float x[NV][VEC], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + l) * VEC;
      Vec<T, VEC> t = {};
      if (on && c < p.cols) t = load_vec<T, VEC>(src + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum += x[i][j] = (float)t.v[j];
    }
    const float mean = mean_of(row_sum<LPR>(sum, lds[0]), p);
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * LPR + l) * VEC < p.cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          x[i][j] -= mean;
          sq = fmaf(x[i][j], x[i][j], sq);
        }
      }
    }
    const float rstd = 1.0f / __builtin_sqrtf(fmaf(row_sum<LPR>(sq, lds[1]), p.inv_cols, p.eps));
    if (!on) continue;
    T* const dst = static_cast<T*>(p.y) + r * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + l) * VEC;
      if (c < p.cols) {
        Vec<T, VEC> t;
#pragma unroll
        for (int j = 0; j < VEC; ++j) t.v[j] = round_to<T>(fmaf(x[i][j] * rstd, w[i][j], b[i][j]));
        store_vec(dst + c, t);
      }
    }
    if (l == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}

template <typename T, int VEC, int LPR, int NV>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256) norm_backward_kernel(NormArgs p) {
  constexpr int kThreads = LPR > 256 ? LPR : 256, kRows = kThreads / LPR;
  __shared__ float lds[2][kThreads / kWave];
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LPR + l) * VEC;
    if (c < p.cols) load_param<T, VEC>(p.weight, p.w32, c, 1.0f, w[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.0f;
  }
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < p.rows; base += (int64_t)gridDim.x * kRows) {
    const int64_t r = base + sub;
    const bool on = r < p.rows;
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
    const T* const grad = static_cast<const T*>(p.d_y) + r * p.cols;
    const float mean = on ? p.mean[r] : 0.0f, rstd = on ? p.rstd[r] : 0.0f;
    float xh[NV][VEC], v[NV][VEC], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + l) * VEC;
      if (on && c < p.cols) {
        const Vec<T, VEC> tx = load_vec<T, VEC>(src + c), tg = load_vec<T, VEC>(grad + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float g = (float)tg.v[j];
          xh[i][j] = ((float)tx.v[j] - mean) * rstd;
          v[i][j] = g * w[i][j];
          dw[i][j] = fmaf(g, xh[i][j], dw[i][j]);
          db[i][j] += g;
          s1 += v[i][j];
          s2 = fmaf(v[i][j], xh[i][j], s2);
        }
      }
    }
    const float m1 = row_sum<LPR>(s1, lds[0]) * p.inv_cols, m2 = row_sum<LPR>(s2, lds[1]) * p.inv_cols;
    if (!on || !p.d_x) continue;
    T* const dst = static_cast<T*>(p.d_x) + r * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + l) * VEC;
      if (c < p.cols) {
        Vec<T, VEC> t;
#pragma unroll
        for (int j = 0; j < VEC; ++j) t.v[j] = round_to<T>(rstd * (v[i][j] - m1 - xh[i][j] * m2));
        store_vec(dst + c, t);
      }
    }
  }
  if (!p.part) return;
  // The rows of a workgroup that ran side by side are summed in their order, then written as one row of partial sums.
  __shared__ float sums[kRows > 1 ? kThreads * VEC * NV : 1];
  float* const out = p.part + (int64_t)blockIdx.x * 2 * p.cols;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if constexpr (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[(sub * NV * VEC + i * VEC + j) * LPR + l] = k ? db[i][j] : dw[i][j];
      __syncthreads();
    }
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + l) * VEC;
        if (c < p.cols) {
          Vec<float, VEC> t;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float s = k ? db[i][j] : dw[i][j];
            if constexpr (kRows > 1)
              for (int q = 1; q < kRows; ++q) s += sums[(q * NV * VEC + i * VEC + j) * LPR + l];
            t.v[j] = s;
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) out[(int64_t)k * p.cols + c + j] = t.v[j];
        }
      }
    }
  }
}

// Rows too long for registers: a workgroup per row, which reads it once per sum.
constexpr int kWideThreads = 1024;

template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(NormArgs p) {
  __shared__ float lds[2][kWideThreads / kWave];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
    float s = 0.0f;
    for (int c = threadIdx.x; c < p.cols; c += kWideThreads) s += (float)src[c];
    const float mean = mean_of(row_sum<kWideThreads>(s, lds[0]), p);
    s = 0.0f;
    for (int c = threadIdx.x; c < p.cols; c += kWideThreads) {
      const float d = (float)src[c] - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.0f / __builtin_sqrtf(fmaf(row_sum<kWideThreads>(s, lds[1]), p.inv_cols, p.eps));
    for (int c = threadIdx.x; c < p.cols; c += kWideThreads) {
      float w[1], b[1];
      load_param<T, 1>(p.weight, p.w32, c, 1.0f, w);
      load_param<T, 1>(p.bias, p.w32, c, 0.0f, b);
      static_cast<T*>(p.y)[r * p.cols + c] = round_to<T>(fmaf(((float)src[c] - mean) * rstd, w[0], b[0]));
    }
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_backward_wide_kernel(NormArgs p) {
  __shared__ float lds[2][kWideThreads / kWave];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* const src = static_cast<const T*>(p.x) + r * p.stride;
    const T* const grad = static_cast<const T*>(p.d_y) + r * p.cols;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < p.cols; c += kWideThreads) {
      float w[1];
      load_param<T, 1>(p.weight, p.w32, c, 1.0f, w);
      const float v = (float)grad[c] * w[0];
      s1 += v;
      s2 = fmaf(v, ((float)src[c] - mean) * rstd, s2);
    }
    const float m1 = row_sum<kWideThreads>(s1, lds[0]) * p.inv_cols;
    const float m2 = row_sum<kWideThreads>(s2, lds[1]) * p.inv_cols;
    for (int c = threadIdx.x; c < p.cols; c += kWideThreads) {
      float w[1];
      load_param<T, 1>(p.weight, p.w32, c, 1.0f, w);
      const float xh = ((float)src[c] - mean) * rstd;
      static_cast<T*>(p.d_x)[r * p.cols + c] = round_to<T>(rstd * ((float)grad[c] * w[0] - m1 - xh * m2));
    }
  }
}

// The workgroups' sums for such rows: a thread per column, the rows in as many runs as there are groups.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(NormArgs p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.cols) return;
  const int64_t per = (p.rows + p.groups - 1) / p.groups;
  const int64_t end = min(p.rows, (blockIdx.y + 1) * per);
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = blockIdx.y * per; r < end; ++r) {
    const float g = (float)static_cast<const T*>(p.d_y)[r * p.cols + c];
    dw = fmaf(g, ((float)static_cast<const T*>(p.x)[r * p.stride + c] - p.mean[r]) * p.rstd[r], dw);
    db += g;
  }
  float* const out = p.part + (int64_t)blockIdx.y * 2 * p.cols;
  out[c] = dw;
  out[(int64_t)p.cols + c] = db;
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
  __syncthreads();
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

// Threads per row and pieces per thread for `pieces` pieces of VEC columns; {0, 0}: too many for registers.
struct Shape {
  int lpr, nv;
};
Shape shape_for(int64_t pieces, int vec) {
  for (int lpr : {8, 16, 32, 64})
    if (pieces <= lpr) return {lpr, 1};
  if (pieces <= 128) return {64, 2};
  if (vec < 8) {
    if (pieces <= 256) return {64, 4};
    for (int lpr : {256, 512, 1024})
      if (pieces <= 4 * lpr) return {lpr, pieces <= 2 * lpr ? 2 : 4};
  } else {
    for (int lpr : {256, 512, 1024})
      if (pieces <= 2 * lpr) return {lpr, pieces <= lpr ? 1 : 2};
  }
  return {0, 0};
}

template <typename T, bool BACKWARD, int VEC, int LPR, int NV>
hipError_t launch_shape(const NormArgs& p, hipStream_t s) {
  constexpr int kThreads = LPR > 256 ? LPR : 256, kRows = kThreads / LPR;
  const int64_t need = (p.rows + kRows - 1) / kRows;
  if (BACKWARD) {
    hipLaunchKernelGGL((norm_backward_kernel<T, VEC, LPR, NV>), dim3((unsigned)std::min<int64_t>(need, p.groups)),
                       dim3(kThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((norm_forward_kernel<T, VEC, LPR, NV>),
                       dim3((unsigned)std::min<int64_t>(need, 256 * 2048 / kThreads)), dim3(kThreads), 0, s, p);
  }
  return hipGetLastError();
}

template <typename T, bool BACKWARD, int VEC>
hipError_t launch_vec(const NormArgs& p, const Shape& sh, hipStream_t s) {
#define PLH_NORM_SHAPE(L, N) \
  if (sh.lpr == L && sh.nv == N) return launch_shape<T, BACKWARD, VEC, L, N>(p, s)
  PLH_NORM_SHAPE(8, 1);
  PLH_NORM_SHAPE(16, 1);
  PLH_NORM_SHAPE(32, 1);
  PLH_NORM_SHAPE(64, 1);
  PLH_NORM_SHAPE(64, 2);
  PLH_NORM_SHAPE(256, 2);
  PLH_NORM_SHAPE(512, 2);
  PLH_NORM_SHAPE(1024, 2);
  if constexpr (VEC == 8) {
    PLH_NORM_SHAPE(256, 1);
  } else {
    PLH_NORM_SHAPE(64, 4);
    PLH_NORM_SHAPE(256, 4);
    PLH_NORM_SHAPE(512, 4);
    PLH_NORM_SHAPE(1024, 4);
  }
#undef PLH_NORM_SHAPE
  return hipErrorInvalidValue;
}

// The widest piece at which every access of a row is aligned.
template <typename T>
int norm_vec(const NormArgs& p) {
  for (int v : {16 / (int)sizeof(T), 4})
    if (p.cols % v == 0 && p.stride % v == 0 && aligned(p.x, v * (int)sizeof(T)) && aligned(p.y, v * (int)sizeof(T)) && aligned(p.d_y, v * (int)sizeof(T)) &&
        aligned(p.d_x, v * (int)sizeof(T)))
      return v;
  return 1;
}

// Workgroups of the backward pass, each with a row of partial sums.
int64_t groups_for(int64_t rows) { return std::max<int64_t>(1, std::min<int64_t>(rows, 1024)); }

template <typename T, bool BACKWARD>
hipError_t launch_norm(NormArgs p, hipStream_t s) {
  const int vec = norm_vec<T>(p);
  const Shape sh = shape_for((p.cols + vec - 1) / vec, vec);
  hipError_t e = hipSuccess;
  const unsigned wide = (unsigned)std::min<int64_t>(p.rows, 1024);
  if (BACKWARD) {
    const bool sums = p.d_weight || p.d_bias;
    if (!sums) p.part = nullptr;
    if (sh.lpr) {
      const int threads = std::max(sh.lpr, 256);
      p.groups = (int)std::min<int64_t>((p.rows + threads / sh.lpr - 1) / (threads / sh.lpr), 1024);
    } else if (p.d_x) {
      hipLaunchKernelGGL(norm_backward_wide_kernel<T>, dim3(wide), dim3(kWideThreads), 0, s, p);
      e = hipGetLastError();
    }
    if (e != hipSuccess) return e;
    if (!sh.lpr && sums) {
      p.groups = (int)std::min<int64_t>(p.rows, 64);
      hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((p.cols + 255) / 256, p.groups), dim3(256), 0, s, p);
      e = hipGetLastError();
    }
    if (e != hipSuccess) return e;
  } else if (!sh.lpr) {
    hipLaunchKernelGGL(norm_forward_wide_kernel<T>, dim3(wide), dim3(kWideThreads), 0, s, p);
    return hipGetLastError();
  }
  if (sh.lpr) {
    if (vec == 8) {
      if constexpr (sizeof(T) == 2) e = launch_vec<T, BACKWARD, 8>(p, sh, s);
    } else if (vec == 4) {
      e = launch_vec<T, BACKWARD, 4>(p, sh, s);
    } else {
      e = launch_vec<T, BACKWARD, 1>(p, sh, s);
    }
    if (e != hipSuccess) return e;
  }
  if (BACKWARD && p.part) {
    hipLaunchKernelGGL(norm_reduce_kernel<T>, dim3((unsigned)((2 * (int64_t)p.cols + 31) / 32)), dim3(1024), 0, s, p);
    e = hipGetLastError();
  }
  return e;
}

int check_norm(const char* what, int dtype, int wdtype, int64_t stride, int64_t rows, int64_t cols, const void* x) noexcept {
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
  return plh::groups_for(rows) * 2 * cols * (int64_t)sizeof(float);
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
