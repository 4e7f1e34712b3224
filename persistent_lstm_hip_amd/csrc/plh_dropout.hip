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

// A thread has the eight elements of one counter, in pieces of 16 bytes.  STREAM: the output is stored past the caches.
template <typename T, bool RESIDUAL, bool STREAM>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs p) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const uint64_t offset = p.offset + (p.offset_dev ? (uint64_t)*p.offset_dev : 0);
  const T* const x = static_cast<const T*>(p.x);
  const T* const res = static_cast<const T*>(p.residual);
  T* const out = static_cast<T*>(p.out);
  const auto masked = [&](uint32_t word, int half, float v) {
    return ((word >> (16 * half)) & 0xFFFFu) >= p.threshold ? v * p.scale : 0.0f;
  };
  const int64_t groups = p.n / 8, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t q = first; q < groups; q += (int64_t)gridDim.x * 256) {
    Vec<T, VEC> vx[8 / VEC], vr[8 / VEC];
#pragma unroll
    for (int i = 0; i < 8 / VEC; ++i) {
      vx[i] = load_vec<T, VEC>(x + q * 8 + i * VEC);
      if (RESIDUAL) vr[i] = load_vec<T, VEC>(res + q * 8 + i * VEC);
    }
    const Words rnd = philox((uint64_t)q, offset, p.seed);
#pragma unroll
    for (int i = 0; i < 8 / VEC; ++i) {
      float y[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        y[j] = masked(rnd.w[(i * VEC + j) / 2], (i * VEC + j) % 2, (float)vx[i].v[j]);
        if (RESIDUAL) y[j] += (float)vr[i].v[j];
      }
      if (STREAM)
        store_vec_stream(out + q * 8 + i * VEC, round_to<T, VEC>(y));
      else
        store_vec(out + q * 8 + i * VEC, round_to<T, VEC>(y));
    }
  }
  const int rest = (int)(p.n % 8);
  if (first < rest) {  // the last elements, a thread each
    const int64_t e = groups * 8 + first;
    const Words rnd = philox((uint64_t)groups, offset, p.seed);
    const uint32_t w01 = first & 2 ? rnd.w[1] : rnd.w[0], w23 = first & 2 ? rnd.w[3] : rnd.w[2];
    float v = masked(first & 4 ? w23 : w01, (int)(first & 1), (float)x[e]);
    if (RESIDUAL) v += (float)res[e];
    out[e] = round_to<T>(v);
  }
}

// Outputs from this size on are larger than the device's L2 caches together and are stored past them (512 x 1000 x 128
// fp16 with a residual 69.4 -> 66.6 us, without 48.2 -> 43.7); what is smaller may be read from there next.
constexpr int64_t kStreamBytes = 32 << 20;

template <typename T>
hipError_t launch_dropout(const DropoutArgs& p, hipStream_t s) {
  // A workgroup per 2048 elements (the loop in the kernel only serves what a grid cannot hold): one pass without a loop
  // takes 69 us where 2048 workgroups that take turns take 78 (as above, with a residual).
  const dim3 grid((unsigned)std::min<int64_t>((p.n + 2047) / 2048, 1 << 23)), block(256);
  const bool stream = p.n * (int64_t)sizeof(T) >= kStreamBytes;
  if (p.residual && stream)
    hipLaunchKernelGGL((dropout_kernel<T, true, true>), grid, block, 0, s, p);
  else if (p.residual)
    hipLaunchKernelGGL((dropout_kernel<T, true, false>), grid, block, 0, s, p);
  else if (stream)
    hipLaunchKernelGGL((dropout_kernel<T, false, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false, false>), grid, block, 0, s, p);
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
