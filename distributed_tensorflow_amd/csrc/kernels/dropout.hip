// Dropout from a counter-based generator: the mask is a function of (seed, step, element index) and is never stored.
//
//   block q = Philox4x32-10(counter = (q, step), key = seed) gives eight 16-bit numbers u, one for each of the elements
//   8q .. 8q + 7;  element i is kept iff u_i >= T, T = round(rate 65536);  y = [residual +] x 65536 / (65536 - T), or 0
//   The scale is the reciprocal of the keep probability that T realises, so the mean is exact for every rate.
//   The gradient is the same map applied to dy.  A dropped element is 0 whatever x holds there (infinity, NaN).
//
// Bound by memory: 16 bits an element, not 32, because ten Philox rounds cost about 20 quarter-rate multiplies a block;
// with four elements a block bf16 data would be bound by those.
// 16384 x 4096 bf16 with residual: 70 us, 5.7 TB/s.  `step` comes from the host, or from a counter in device
// memory, so that a replayed graph draws new masks; the value used is stored for the backward pass.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "token_ops.h"

namespace {
struct DropArgs {
  const void* x; const void* res; void* y; const long long* step_ptr; long long* used;
  int64_t n; uint64_t seed, step; unsigned thr; float scale;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
  constexpr int PER16 = 16 / sizeof(T);
  const uint64_t step = a.step + (a.step_ptr ? (uint64_t)*a.step_ptr : 0);
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x, i0 = q * 8;
  if (q == 0 && a.used) *a.used = (long long)step;
  if (i0 >= a.n) return;
  const T* const x = static_cast<const T*>(a.x) + i0;
  const T* const r = a.res ? static_cast<const T*>(a.res) + i0 : nullptr;
  T* const y = static_cast<T*>(a.y) + i0;
  const bool full = VEC && i0 + 8 <= a.n;
  const int cnt = a.n - i0 < 8 ? (int)(a.n - i0) : 8;
  float v[8 / PER16][PER16], z[8 / PER16][PER16];
#pragma unroll
  for (int k = 0; k < 8 / PER16; ++k) {
    if (full) {
      TkVec<T, PER16>::load(x + k * PER16, v[k]);
      if (r) TkVec<T, PER16>::load(r + k * PER16, z[k]);
    } else {
#pragma unroll
      for (int e = 0; e < PER16; ++e) {
        v[k][e] = k * PER16 + e < cnt ? tk_get(x + k * PER16 + e) : 0.f;
        z[k][e] = r && k * PER16 + e < cnt ? tk_get(r + k * PER16 + e) : 0.f;
      }
    }
  }
  uint32_t c[4] = {(uint32_t)q, (uint32_t)((uint64_t)q >> 32), (uint32_t)step, (uint32_t)(step >> 32)};
  tk_philox(c, (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
#pragma unroll
  for (int k = 0; k < 8 / PER16; ++k) {
#pragma unroll
    for (int e = 0; e < PER16; ++e) {
      const int i = k * PER16 + e;
      const unsigned u = (c[i >> 1] >> (16 * (i & 1))) & 0xffffu;
      v[k][e] = u >= a.thr ? v[k][e] * a.scale : 0.f;
      if (r) v[k][e] += z[k][e];
    }
    if (full) {
      TkVec<T, PER16>::store(y + k * PER16, v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < PER16; ++e)
        if (k * PER16 + e < cnt) tk_put(y + k * PER16 + e, v[k][e]);
    }
  }
}
}  // namespace

// n dense elements; step = *step_ptr (if given) + step; *used (if given) = the step used.  y may be x or res.
DTF_EXPORT int dtf_dropout(const void* x, const void* res, void* y, int64_t n, int dtype, double rate, uint64_t seed, uint64_t step,
                           const long long* step_ptr, long long* used, hipStream_t s) {
  if (!(rate >= 0.0 && rate <= 1.0) || (dtype != TK_F32 && dtype != TK_BF16)) return DTF_ERR_ARG;
  if (n < 0 || n >= (1ll << 35) - 4096) return DTF_ERR_SHAPE;         // fewer than 2^32 threads
  if (n > 0 && (!x || !y)) return DTF_ERR_ARG;
  if (n == 0 && !used) return DTF_OK;
  const unsigned thr = (unsigned)__builtin_rint(rate * 65536.0);     // ties to even, like Python's round
  const DropArgs a = {x, res, y, step_ptr, used, n, seed, step, thr, thr < 65536u ? (float)(65536.0 / (65536u - thr)) : 0.f};
  const dim3 g((unsigned)std::max<int64_t>(1, (n + 2047) / 2048)), b(256);
  const bool v = dtf_aligned16(x) && dtf_aligned16(y) && (!res || dtf_aligned16(res));
  if (dtype == TK_BF16) {
    if (v) hipLaunchKernelGGL((dropout_kernel<unsigned short, true>), g, b, 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<unsigned short, false>), g, b, 0, s, a);
  } else {
    if (v) hipLaunchKernelGGL((dropout_kernel<float, true>), g, b, 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<float, false>), g, b, 0, s, a);
  }
  return dtf_check_launch();
}
