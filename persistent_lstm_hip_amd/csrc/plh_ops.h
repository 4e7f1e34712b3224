// plh_ops.h -- what the block operators (plh_scan.hip, plh_norm.hip, plh_dropout.hip) share: element types, vector
// loads and stores, the logistic function, and the host's error reporting.
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

// N consecutive elements, moved with one load or store of N * sizeof(T) bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) {
  *reinterpret_cast<Vec<T, N>*>(p) = v;
}

// v rounded to T as an fp32 value.  (Left alone, the compiler may fold the operation that made v into the conversion,
// in some variants of a kernel and not in others, which then differ in a last place now and then.)
template <typename T>
__device__ __forceinline__ T round_to(float v) {
  if constexpr (sizeof(T) < sizeof(float)) asm("" : "+v"(v));
  return (T)v;
}

constexpr float kOpLog2e = 1.4426950408889634f;

// The logistic function and its complement, s = 1 / (1 + e) and 1 - s = e s with e = 2^min(-z log2 e, 126): the
// complement keeps its relative precision where s is close to 1, and the cap keeps e s from being inf * 0 (it moves s
// by less than 2^-126).  The minimum returns NaN for a NaN argument.
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

template <typename T>
inline bool aligned(const void* p, int n) {
  return (reinterpret_cast<uintptr_t>(p) % (sizeof(T) * n)) == 0;
}

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
