// Launch and dispatch conditions of the 8-wave bf16 GEMM (kernel, layout and schedule: gemm_pingpong.h), and the summing
// pass of its split-K weight gradient.
#include <cstdlib>

#include "gemm_pingpong.h"

// Shapes this kernel takes: bf16, M, N and K multiples of 8 (16-byte chunks of operands and outputs), K at least
// 256, the transposed mask for the backward epilogue, outputs that take 16-byte stores.  Whether it PAYS (enough
// 256x256 blocks to fill the chip, little waste at ragged edges) is the caller's decision.
// dst[i] = sum over the splits, in split order, of the partial weight gradients (ld = ldc: M * ldc floats per split,
// a multiple of 4) and partial bias gradients
__global__ __launch_bounds__(256) void splitk_sum_kernel(float* __restrict__ dst, const float* __restrict__ ws, long n4, long stride,
                                                         float* __restrict__ bias_dst, const float* __restrict__ bias_ws, int N, int S) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i < n4) {
    f32x4 acc = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(ws) + i);
    for (int s = 1; s < S; ++s) {
      const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(ws + (size_t)s * stride) + i);
      acc[0] += v[0]; acc[1] += v[1]; acc[2] += v[2]; acc[3] += v[3];
    }
    reinterpret_cast<f32x4*>(dst)[i] = acc;
  } else if (bias_dst && i - n4 < N) {
    const int c = (int)(i - n4);
    float acc = bias_ws[c];
    for (int s = 1; s < S; ++s) acc += bias_ws[(size_t)s * N + c];
    bias_dst[c] = acc;
  }
}

bool dtf_gemm_pingpong_takes(const DtfGemmArgs& a) {
  if (a.dtype != 1 || (a.M & 7) || (a.N & 7) || (a.K & 7) || a.K < 256) return false;
  if (a.ksplit > 1) {
    if (a.epilogue != EPI_WGRAD || a.opt_p || !a.split_ws || (a.bias_out && !a.split_bias_ws)) return false;
    if (a.ksplit > 16 || a.K / a.ksplit < 256 || (reinterpret_cast<uintptr_t>(a.split_ws) & 15)) return false;
    if (a.ldc != a.N) return false;           // the summing pass treats C and each partial as M * N contiguous floats
  }
  if (a.epilogue == EPI_BWD && (!a.maskT || (a.ldmaskt & 3))) return false;
  if ((reinterpret_cast<uintptr_t>(a.C) & 15) || (a.ldc & (a.epilogue == EPI_WGRAD ? 3 : 7))) return false;
  if (a.Ct && ((a.ldct & 7) || (reinterpret_cast<uintptr_t>(a.Ct) & 15))) return false;
  if (a.maskT && (reinterpret_cast<uintptr_t>(a.maskT) & 7)) return false;
  if (a.opt_p) {
    if (a.epilogue != EPI_WGRAD || (a.opt_m == nullptr) != (a.opt_v == nullptr)) return false;
    if ((reinterpret_cast<uintptr_t>(a.opt_p) & 15) || (a.opt_m && ((reinterpret_cast<uintptr_t>(a.opt_m) | reinterpret_cast<uintptr_t>(a.opt_v)) & 15))) return false;
    if (a.opt_w && (reinterpret_cast<uintptr_t>(a.opt_w) & 7)) return false;
    if (a.opt_wt && ((reinterpret_cast<uintptr_t>(a.opt_wt) & 15) || (a.ldwt & 7) || a.ldwt < a.M)) return false;
  }
  return true;
}

int dtf_gemm_pingpong_launch(const DtfGemmArgs& a_in, hipStream_t s) {
  if (!dtf_gemm_pingpong_takes(a_in)) return DTF_ERR_SHAPE;
#ifdef DTF_STAMPS
  static int skip = -1;
  if (skip < 0) {
    const char* e = getenv("DTF_GEMM_SKIP_STORES");
    skip = e ? atoi(e) & 3 : 0;
  }
  DtfGemmArgs a = a_in;
  a.pad_ = skip;
#else
  const DtfGemmArgs& a = a_in;
#endif
  const int split = a.ksplit > 1 ? a.ksplit : 1;
  dim3 grid(((a.M + 255) >> 8) * ((a.N + 255) >> 8) * split), block(512);
  switch (a.epilogue) {
    case EPI_FWD: hipLaunchKernelGGL((gemm_pp_kernel<EPI_FWD, DtfGemmArgs>), grid, block, 0, s, a); break;
    case EPI_BWD: hipLaunchKernelGGL((gemm_pp_kernel<EPI_BWD, DtfGemmArgs>), grid, block, 0, s, a); break;
    case EPI_WGRAD:
      if (a.opt_p) hipLaunchKernelGGL((gemm_pp_kernel<EPI_WGRAD_OPT, DtfGemmArgs>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((gemm_pp_kernel<EPI_WGRAD, DtfGemmArgs>), grid, block, 0, s, a);
      break;
    default: return DTF_ERR_ARG;
  }
  if (split > 1) {
    const long n4 = (long)a.M * a.ldc / 4;
    const long threads = n4 + (a.bias_out ? a.N : 0);
    hipLaunchKernelGGL(splitk_sum_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, static_cast<float*>(a.C),
                       a.split_ws, n4, (long)a.M * a.ldc, a.bias_out, a.split_bias_ws, a.N, split);
  }
  return dtf_check_launch();
}
