// plh_dropout.hip -- dropout from a counter-based generator, with an optional residual added in the same pass.
//
//   out[e] = residual[e] + (r(e) >= threshold ? x[e] * 65536 / (65536 - threshold) : 0)
//
// r(e) is 16 bits of Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", SC 2011): a bijection of a 128-bit counter under a 64-bit key in ten rounds of two 32 x 32 -> 64 bit products.
// One call of it serves eight elements, so the mask is a function of (seed, offset, e) and is computed again where the
// gradient needs it.  Sixteen bits per element keep the generator, at ten rounds per eight elements, below the time of
// the memory traffic; probabilities are multiples of 2^-16 and the scale is that of the multiple, so that the mean is
// kept exactly.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "plh_ops.h"

namespace plh {
namespace {

struct DropoutArgs {
  const void *x, *residual;
  void* out;
  int64_t n;
  uint32_t threshold;
  float scale;
  uint64_t seed, offset;
  const int64_t* offset_dev;
};

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t ctr, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)ctr, c1 = (uint32_t)(ctr >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// A thread has the eight elements of one counter, in pieces of VEC.
template <typename T, int VEC, bool RESIDUAL>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs p) {
  const uint64_t offset = p.offset + (p.offset_dev ? (uint64_t)*p.offset_dev : 0);
  const T* const x = static_cast<const T*>(p.x);
  const T* const res = static_cast<const T*>(p.residual);
  T* const out = static_cast<T*>(p.out);
  const int64_t groups = (p.n + 7) / 8;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < groups; q += (int64_t)gridDim.x * 256) {
    const int64_t e = q * 8;
    const int live = (int)min<int64_t>(8, p.n - e);
    T vx[8], vr[8];
    if (live == 8) {
#pragma unroll
      for (int i = 0; i < 8; i += VEC) {
        const Vec<T, VEC> a = load_vec<T, VEC>(x + e + i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) vx[i + j] = a.v[j];
        if (RESIDUAL) {
          const Vec<T, VEC> b = load_vec<T, VEC>(res + e + i);
#pragma unroll
          for (int j = 0; j < VEC; ++j) vr[i + j] = b.v[j];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        vx[i] = i < live ? x[e + i] : (T)0.0f;
        vr[i] = RESIDUAL && i < live ? res[e + i] : (T)0.0f;
      }
    }
    const Words rnd = philox((uint64_t)q, offset, p.seed);
    T y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t r = (rnd.w[i / 2] >> (16 * (i % 2))) & 0xFFFFu;
      float v = r >= p.threshold ? (float)vx[i] * p.scale : 0.0f;
      if (RESIDUAL) v += (float)vr[i];
      y[i] = round_to<T>(v);
    }
    if (live == 8) {
#pragma unroll
      for (int i = 0; i < 8; i += VEC) {
        Vec<T, VEC> a;
#pragma unroll
        for (int j = 0; j < VEC; ++j) a.v[j] = y[i + j];
        store_vec(out + e + i, a);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < live) out[e + i] = y[i];
    }
  }
}

template <typename T>
hipError_t launch_dropout(const DropoutArgs& p, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const unsigned grid = (unsigned)std::min<int64_t>((p.n + 2047) / 2048, 256 * 8);
  const bool wide = aligned(p.x, 16) && aligned(p.residual, 16) && aligned(p.out, 16);
  if (wide && p.residual)
    hipLaunchKernelGGL((dropout_kernel<T, V, true>), dim3(grid), dim3(256), 0, s, p);
  else if (wide)
    hipLaunchKernelGGL((dropout_kernel<T, V, false>), dim3(grid), dim3(256), 0, s, p);
  else if (p.residual)
    hipLaunchKernelGGL((dropout_kernel<T, 1, true>), dim3(grid), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((dropout_kernel<T, 1, false>), dim3(grid), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace plh

extern "C" int plh_dropout_add(int dtype, const void* x, const void* residual, void* out, int64_t n, int threshold,
                               uint64_t seed, uint64_t offset, const int64_t* offset_dev, void* stream) {
  const char* const what = "dropout_add";
  if (dtype != PLH_F16 && dtype != PLH_BF16 && dtype != PLH_F32)
    return plh::op_error(PLH_ERR_INVALID, what, "dtype must be PLH_F16, PLH_BF16 or PLH_F32");
  if (n < 0) return plh::op_error(PLH_ERR_INVALID, what, "n must be non-negative");
  if (threshold < 0 || threshold > 65536) return plh::op_error(PLH_ERR_INVALID, what, "threshold must lie in [0, 65536]");
  if (n == 0) return PLH_OK;
  if (!x || !out) return plh::op_error(PLH_ERR_INVALID, what, "x and out are required");
  plh::DropoutArgs p = {};
  p.x = x, p.residual = residual, p.out = out, p.n = n;
  p.threshold = (uint32_t)threshold;
  p.scale = threshold < 65536 ? 65536.0f / (float)(65536 - threshold) : 0.0f;  // (65536: nothing is kept)
  p.seed = seed, p.offset = offset, p.offset_dev = offset_dev;
  hipError_t e = hipSuccess;
  plh::with_dtype(dtype, [&](auto zero) { e = plh::launch_dropout<decltype(zero)>(p, (hipStream_t)stream); });
  return e == hipSuccess ? PLH_OK : plh::op_error(e, what);
}
