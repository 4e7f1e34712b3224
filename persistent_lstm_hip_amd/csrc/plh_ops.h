// plh_ops.h -- what the block operators (plh_scan.hip, plh_norm.hip, plh_dropout.hip, plh_conv.hip, plh_selective.hip,
// plh_clip.hip) share: element types, vector loads and stores, the logistic function, column sums, and the host's error
// reporting.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/persistent_lstm_hip.h"

namespace plh {

// Records the calling thread's error message (plh_last_error) and returns `code`.  Defined in plh_capi.hip.
int op_error(int code, const char* what, const char* msg) noexcept;
int op_error(hipError_t e, const char* what) noexcept;

namespace {

constexpr int kWave = 64;

// N consecutive elements, moved with one load or store of N * sizeof(T) bytes.  The address needs an element's
// alignment only: gfx950 takes wide global accesses at any (element) address, so odd row lengths and strides cost the
// lines that they straddle and no narrower instruction.
template <typename T, int N>
struct Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  Vec<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) {
  __builtin_memcpy(p, &v, sizeof(v));
}

// A store of 16 bytes that is not to be kept in the caches.
template <typename T, int N>
__device__ __forceinline__ void store_vec_stream(T* p, const Vec<T, N>& v) {
  static_assert(sizeof(v) == 16, "16 bytes");
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef u32x4 u32x4_at_any __attribute__((aligned(2)));
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4_at_any*>(p));
}

// Barrier that orders LDS traffic only: global loads and stores stay in flight across it (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Values rounded to T as fp32 values.  (Left alone, the compiler may fold the operation that made a value into its
// conversion, in some variants of a kernel and not in others, which then differ in a last place now and then.)
template <typename T>
__device__ __forceinline__ T round_to(float v) {
  if constexpr (sizeof(T) < sizeof(float)) asm("" : "+v"(v));
  return (T)v;
}
// The same for a vector, with one conversion instruction for two values of 16 bits.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> round_to(const float (&v)[N]) {
  Vec<T, N> r;
  if constexpr (sizeof(T) < sizeof(float) && N % 2 == 0) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      f32x2 p = {v[j], v[j + 1]};
      asm("" : "+v"(p));
      const t2 q = __builtin_convertvector(p, t2);
      r.v[j] = q[0], r.v[j + 1] = q[1];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) r.v[j] = round_to<T>(v[j]);
  }
  return r;
}

constexpr float kOpLog2e = 1.4426950408889634f;

// The logistic function and its complement, s = 1 / (1 + e) and 1 - s = e s with e = 2^min(-z log2 e, 126): the
// complement keeps its relative precision where s is close to 1, and the cap keeps e s from being inf * 0 (it moves s
// by less than 2^-126).  The minimum returns NaN for a NaN argument.  The exponent is one rounded product, so that e, and
// with it the smaller of the two, is within (8 + 1.5 |z|) 2^-24 of its value, relative; absolutely both are within 8 2^-24.
__device__ __forceinline__ void logistic_fast(float z, float& s, float& not_s) {
  const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(z * -kOpLog2e, 126.0f));
  s = __builtin_amdgcn_rcpf(1.0f + e);
  not_s = e * s;
}
// The same for values that are multiplied with each other many times over: v_rcp_f32 alone is off by up to one unit
// in the last place, one step of Newton's iteration rounds it.
__device__ __forceinline__ void logistic(float z, float& s, float& not_s) {
  const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(z * -kOpLog2e, 126.0f));
  const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
  s = fmaf(fmaf(-d, r, 1.0f), r, r);
  not_s = e * s;
}
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -kOpLog2e));
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

// The slab of a launch's workgroup i of n.  Workgroups go round the eight XCDs in turn; here each XCD gets neighbouring
// slabs, so that a cache line that two slabs share is read into one L2 (33 x 1001 x 333 fp16, no slab aligned: forward
// 47.7 -> 40.2 us, backward 79.4 -> 68.2).
__device__ __forceinline__ unsigned slab_of(unsigned i, unsigned n) {
  const unsigned per = n / 8;
  return i < per * 8 ? (i % 8) * per + i / 8 : i;
}

// Column sums of partial results [rows][cols] in a fixed order, to up to three outputs that share the columns: output k has
// those from begin[k] to begin[k + 1], of T, or fp32 (out32); null: not wanted.  No rows: zeros.
struct ColumnSums {
  const float* part;
  int64_t rows, cols;
  bool out32;
  void* out[3];
  int64_t begin[4];
};

// 32 threads per column, whose rows are 32 apart.
template <typename T>
__global__ void __launch_bounds__(1024) column_sums_kernel(ColumnSums p) {
  __shared__ float lds[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const int q = threadIdx.x / 32;
  float s = 0.0f;
  if (c < p.cols) {
#pragma unroll 8
    for (int64_t r = q; r < p.rows; r += 32) s += p.part[r * p.cols + c];
  }
  lds[q][threadIdx.x % 32] = s;
  lds_barrier();
  if (q != 0 || c >= p.cols) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += lds[i][threadIdx.x];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (c < p.begin[k] || c >= p.begin[k + 1] || !p.out[k]) continue;
    if (p.out32)
      static_cast<float*>(p.out[k])[c - p.begin[k]] = s;
    else
      static_cast<T*>(p.out[k])[c - p.begin[k]] = round_to<T>(s);
  }
}

template <typename T>
inline hipError_t launch_column_sums(const ColumnSums& p, hipStream_t s) {
  hipLaunchKernelGGL(column_sums_kernel<T>, dim3((unsigned)((p.cols + 31) / 32)), dim3(1024), 0, s, p);
  return hipGetLastError();
}

// silu(v) = v sigmoid(v) and its derivative; minus infinity gives zero, not inf * 0.
__device__ __forceinline__ float silu(float v) {
  return __builtin_elementwise_maximum(v, -3e38f) * sigmoid(v);
}
__device__ __forceinline__ float silu_slope(float v) {
  const float s = sigmoid(v), f = __builtin_elementwise_minimum(__builtin_elementwise_maximum(v, -3e38f), 3e38f);
  return s * fmaf(f, 1.0f - s, 1.0f);
}

__device__ __forceinline__ void silu(float v, float& value, float& slope) {
  const float s = sigmoid(v), low = __builtin_elementwise_maximum(v, -3e38f);
  value = low * s;
  slope = s * fmaf(__builtin_elementwise_minimum(low, 3e38f), 1.0f - s, 1.0f);
}

inline bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// Calls f with a value of the element type that `dtype` names; false if it names none.
template <typename F>
inline bool with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case PLH_F16: f(_Float16()); return true;
    case PLH_BF16: f(__bf16()); return true;
    case PLH_F32: f(float()); return true;
    default: return false;
  }
}

}  // namespace
}  // namespace plh
