// Launch and dispatch of the tiled GEMMs (register-staged 4-wave kernels: gemm_tiled.h; large aligned bf16 products:
// gemm_pingpong.hip), and the streaming helpers of the wide pipeline.
#include <cstdlib>

#include "gemm_tiled.h"

template <typename T, int TI, int TJ>
static int launch_tiled_as(const DtfGemmArgs& a, hipStream_t s) {
  const int tiles = dtf_cdiv(a.M, 32 * TI) * dtf_cdiv(a.N, 32 * TJ);
  dim3 grid(tiles), block(256);
  switch (a.epilogue) {
    case EPI_FWD: hipLaunchKernelGGL((gemm_tiled_kernel<T, EPI_FWD, TI, TJ, DtfGemmArgs>), grid, block, 0, s, a); break;
    case EPI_BWD: hipLaunchKernelGGL((gemm_tiled_kernel<T, EPI_BWD, TI, TJ, DtfGemmArgs>), grid, block, 0, s, a); break;
    case EPI_WGRAD: hipLaunchKernelGGL((gemm_tiled_kernel<T, EPI_WGRAD, TI, TJ, DtfGemmArgs>), grid, block, 0, s, a); break;
    default: return DTF_ERR_ARG;
  }
  return dtf_check_launch();
}

// gemm_pingpong.hip: 8-wave 256x256 kernel for large aligned bf16 products
bool dtf_gemm_pingpong_takes(const DtfGemmArgs& a);
int dtf_gemm_pingpong_launch(const DtfGemmArgs& a, hipStream_t s);
static int g_pingpong_mode = -1;      // -1 = unread, 0 = never, 1 = whenever the shape allows, 2 = by problem size (DTF_GEMM_PINGPONG)

static int g_big_tile_mode = -1;      // -1 = by problem size, 0 = never, 1 = always (DTF_GEMM_BIG_TILE)

template <typename T>
static int launch_tiled(const DtfGemmArgs& a, hipStream_t s) {
  if (g_big_tile_mode < 0) {
    const char* e = getenv("DTF_GEMM_BIG_TILE");
    g_big_tile_mode = e ? (e[0] == '1' ? 1 : (e[0] == '0' ? 0 : 2)) : 2;
  }
  // 256x256 blocks pay off once they fill the chip (one block per CU, 256 CUs) and waste little at the edges
  const long big_tiles = (long)dtf_cdiv(a.M, 256) * dtf_cdiv(a.N, 256);
  const bool fits = big_tiles >= 192 && (a.M % 256 == 0 || a.M >= 2048) && (a.N % 256 == 0 || a.N >= 2048);
  // measured at 8192x4096x4096 bf16: forward 714 -> 787, weight gradient 778 -> 901 TFLOP/s; the backward epilogue
  // (one mask element per output element) is not overlapped by a second resident workgroup any more: 663 -> 587,
  // so it keeps the 128x128 blocks
  const bool suited = a.epilogue != EPI_BWD || a.maskT != nullptr;
  if (g_pingpong_mode < 0) {
    const char* e = getenv("DTF_GEMM_PINGPONG");
    g_pingpong_mode = e ? (e[0] == '1' ? 1 : (e[0] == '0' ? 0 : 2)) : 2;
  }
  if (a.opt_p || a.ksplit > 1)      // folded optimizer, split-K: 8-wave kernel only, and the caller asked for exactly that
    return (sizeof(T) == 2 && dtf_gemm_pingpong_takes(a)) ? dtf_gemm_pingpong_launch(a, s) : (int)DTF_ERR_SHAPE;
  if (sizeof(T) == 2 && g_pingpong_mode && dtf_gemm_pingpong_takes(a) && (g_pingpong_mode == 1 || fits))
    return dtf_gemm_pingpong_launch(a, s);
  if (sizeof(T) == 2 && (g_big_tile_mode == 1 || (g_big_tile_mode == 2 && fits && suited))) return launch_tiled_as<T, 8, 8>(a, s);
  return launch_tiled_as<T, 4, 4>(a, s);
}

// Kernel selection for tests and tools: 0 = never, 1 = whenever the shape allows, 2 = by problem size, -1 = leave as is
// (the defaults come from DTF_GEMM_BIG_TILE / DTF_GEMM_PINGPONG, read on first use).
DTF_EXPORT void dtf_gemm_set_modes(int big_tile, int pingpong) {
  if (big_tile >= 0) g_big_tile_mode = big_tile;
  if (pingpong >= 0) g_pingpong_mode = pingpong;
}

DTF_EXPORT int dtf_gemm_tiled(const DtfGemmArgs* a, hipStream_t s) {
  if (!a || !a->A || !a->B || !a->C) return DTF_ERR_ARG;
  if (a->M <= 0 || a->N <= 0 || a->K <= 0) return DTF_ERR_SHAPE;
  const int per16 = a->dtype == 1 ? 8 : 4;
  if (a->dtype != 0 && a->dtype != 1) return DTF_ERR_ARG;
  // 16-byte staging loads: K and both leading dimensions in whole 16-byte chunks, aligned bases
  if (a->K % per16 || a->lda % per16 || a->ldb % per16) return DTF_ERR_ALIGN;
  if (!dtf_aligned16(a->A) || !dtf_aligned16(a->B)) return DTF_ERR_ALIGN;
  if (a->lda < a->K || a->ldb < a->K || a->ldc < a->N) return DTF_ERR_SHAPE;
  const uint64_t es = a->dtype == 1 ? 2 : 4;
  if (a->a_bytes == 0 || a->b_bytes == 0 || a->a_bytes >= kOOB || a->b_bytes >= kOOB) return DTF_ERR_SHAPE;
  if (((uint64_t)(a->M - 1) * a->lda + a->K) * es > a->a_bytes) return DTF_ERR_SHAPE;
  if (((uint64_t)(a->N - 1) * a->ldb + a->K) * es > a->b_bytes) return DTF_ERR_SHAPE;
  if (a->epilogue == EPI_BWD && (!a->mask || a->ldmask < a->N)) return DTF_ERR_ARG;
  if (a->maskT && (a->ldmaskt < a->M || !dtf_aligned16(a->maskT))) return DTF_ERR_SHAPE;
  if (a->Ct && a->ldct < a->M) return DTF_ERR_SHAPE;
  if (a->C32 && a->ldc32 < a->N) return DTF_ERR_SHAPE;
  if (a->epilogue == EPI_WGRAD && (a->Ct || a->C32)) return DTF_ERR_ARG;
  if (a->opt_p && a->epilogue != EPI_WGRAD) return DTF_ERR_ARG;
  return a->dtype == 1 ? launch_tiled<unsigned short>(*a, s) : launch_tiled<unsigned int>(*a, s);
}

// --------------------------------------------------------------------------------------
// helpers of the wide pipeline (pure streaming kernels)
// --------------------------------------------------------------------------------------
// dst[i] = src[rows[i]] converted to T, plus the transposed copy dstT[c][i]  (batch gather for layer 1,
// compute copies of the weights).  64x64 tiles: 16-byte global loads, the tile held in LDS in the output
// type, straight and transposed copies written as 8-byte (bf16) / 16-byte (fp32) pieces of 4 elements.
template <typename T>
__global__ __launch_bounds__(256) void gather_cast_transpose_kernel(const float* __restrict__ src, const int* __restrict__ rows,
                                                                    T* __restrict__ dst, T* __restrict__ dstT, int M, int N,
                                                                    int lds_, int ldd, int ldt) {
  __shared__ T tile[64][65];
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;   // 16 x 16 threads, 4 elements each per pass
  const bool vec_in = ((lds_ & 3) == 0) && (((uintptr_t)src & 15) == 0);
  const bool vec_out = dst && ((ldd & 3) == 0) && (((uintptr_t)dst & 15) == 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = ty + 16 * i, r = r0 + rr, c = c0 + 4 * tx;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < M) {
      const size_t base = (size_t)(rows ? rows[r] : r) * lds_ + c;
      if (vec_in && c + 3 < N) {
        const float4 q = *reinterpret_cast<const float4*>(src + base);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < N) v[j] = src[base + j];
      }
    }
    T o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j] = sizeof(T) == 2 ? (T)f2bf(v[j]) : (T)__float_as_uint(v[j]);
      tile[rr][4 * tx + j] = o[j];
    }
    if (dst && r < M) {
      T* d = dst + (size_t)r * ldd + c;
      if (vec_out && c + 3 < N) {
        if (sizeof(T) == 2) *reinterpret_cast<uint2*>(d) = make_uint2((unsigned)o[0] | ((unsigned)o[1] << 16), (unsigned)o[2] | ((unsigned)o[3] << 16));
        else *reinterpret_cast<uint4*>(d) = make_uint4((unsigned)o[0], (unsigned)o[1], (unsigned)o[2], (unsigned)o[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < N) d[j] = o[j];
      }
    }
  }
  __syncthreads();
  if (!dstT) return;
  const bool vec_t = ((ldt & 3) == 0) && (((uintptr_t)dstT & 15) == 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int cc = ty + 16 * i, c = c0 + cc, r = r0 + 4 * tx;   // output row c, 4 consecutive source rows
    if (c >= N) continue;
    T o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = tile[4 * tx + j][cc];
    T* d = dstT + (size_t)c * ldt + r;
    if (vec_t && r + 3 < M) {
      if (sizeof(T) == 2) *reinterpret_cast<uint2*>(d) = make_uint2((unsigned)o[0] | ((unsigned)o[1] << 16), (unsigned)o[2] | ((unsigned)o[3] << 16));
      else *reinterpret_cast<uint4*>(d) = make_uint4((unsigned)o[0], (unsigned)o[1], (unsigned)o[2], (unsigned)o[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r + j < M) d[j] = o[j];
    }
  }
}

// dstT[c][r] = src[r][c] for 2-byte elements (the transposed compute copy of weights whose straight copy the
// weight-gradient epilogue has just written).  64x64 tiles through LDS, 16-byte global accesses on both sides.
__global__ __launch_bounds__(256) void transpose16_kernel(const unsigned short* __restrict__ src, unsigned short* __restrict__ dstT,
                                                          int M, int N, int lds_, int ldt) {
  __shared__ unsigned short tile[64][72];           // 144-byte rows: 16-byte aligned, column reads spread over banks
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int id = t + 256 * i, rr = id >> 3, ch = id & 7;          // row, 16-byte chunk of 8 columns
    u32x4 v = {0u, 0u, 0u, 0u};
    if (r0 + rr < M && c0 + ch * 8 < N) v = *reinterpret_cast<const u32x4*>(src + (size_t)(r0 + rr) * lds_ + c0 + ch * 8);
    *reinterpret_cast<u32x4*>(&tile[rr][ch * 8]) = v;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int id = t + 256 * i, cc = id >> 3, ch = id & 7;          // output row (a source column), chunk of 8 source rows
    if (c0 + cc >= N || r0 + ch * 8 >= M) continue;
    unsigned short e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = tile[ch * 8 + k][cc];
    u32x4 v = {(unsigned)e[0] | ((unsigned)e[1] << 16), (unsigned)e[2] | ((unsigned)e[3] << 16),
               (unsigned)e[4] | ((unsigned)e[5] << 16), (unsigned)e[6] | ((unsigned)e[7] << 16)};
    *reinterpret_cast<u32x4*>(dstT + (size_t)(c0 + cc) * ldt + r0 + ch * 8) = v;
  }
}

DTF_EXPORT int dtf_transpose16(const void* src, void* dstT, int M, int N, int lds_, int ldt, hipStream_t s) {
  if (!src || !dstT) return DTF_ERR_ARG;
  if (M <= 0 || N <= 0 || (M & 7) || (N & 7) || lds_ < N || ldt < M || (lds_ & 7) || (ldt & 7)) return DTF_ERR_SHAPE;
  if (!dtf_aligned16(src) || !dtf_aligned16(dstT)) return DTF_ERR_ALIGN;
  if (dtf_cdiv(M, 64) > 65535) return DTF_ERR_SHAPE;
  hipLaunchKernelGGL(transpose16_kernel, dim3(dtf_cdiv(N, 64), dtf_cdiv(M, 64)), dim3(256), 0, s,
                     static_cast<const unsigned short*>(src), static_cast<unsigned short*>(dstT), M, N, lds_, ldt);
  return dtf_check_launch();
}

DTF_EXPORT int dtf_gather_cast_transpose(const float* src, const int* rows, void* dst, void* dstT, int M, int N, int lds_,
                                         int ldd, int ldt, int dtype, hipStream_t s) {
  if (!src || (!dst && !dstT)) return DTF_ERR_ARG;
  if (M <= 0 || N <= 0 || lds_ < N || (dst && ldd < N) || (dstT && ldt < M)) return DTF_ERR_SHAPE;
  if (dtf_cdiv(M, 64) > 65535) return DTF_ERR_SHAPE;
  dim3 grid(dtf_cdiv(N, 64), dtf_cdiv(M, 64)), block(256);
  if (dtype == 1)
    hipLaunchKernelGGL(gather_cast_transpose_kernel<unsigned short>, grid, block, 0, s, src, rows, (unsigned short*)dst,
                       (unsigned short*)dstT, M, N, lds_, ldd, ldt);
  else if (dtype == 0)
    hipLaunchKernelGGL(gather_cast_transpose_kernel<unsigned int>, grid, block, 0, s, src, rows, (unsigned int*)dst,
                       (unsigned int*)dstT, M, N, lds_, ldd, ldt);
  else
    return DTF_ERR_ARG;
  return dtf_check_launch();
}
