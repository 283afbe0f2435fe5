// Softmax cross entropy over a large vocabulary without keeping the logits: z = X W^T + b, X [N tokens, D], W [V, D].
//
//   forward    lse_r = log sum_c exp z_rc;   loss_r = lse_r - z_r,label;   hit_r: label is the first maximum of the row
//   backward   dz_rc = (exp(z_rc - lse_r) - [c = label_r]) g_r;   dX = dz W;   dW = dz^T X;   db_c = sum_r dz_rc
//
// Forward: one GEMM whose epilogue reduces each row of a wave's 64-column strip to (maximum, sum of exponentials) and
// picks the label's logit on the way; a join over the strips gives lse, loss and hits.  8 bytes a strip and row leave the
// chip instead of 256 of logits.
// Backward: the vocabulary is cut into pieces; for each piece the same GEMM is run again and its epilogue writes dz in the
// operands' type, once as [N, piece] and once transposed, which are the operands of the two products dX += dz W and
// dW = dz^T X (all products in the one form A[M,K] . B[N,K]^T of the tiled GEMMs).  The work is 8 N V D operations instead
// of the 6 N V D of a program that stores the logits: at N = 8192, V = 131072 the fp32 logits would be 4 GB to write and
// read again, 2.1 GB of bf16 dz per step go through a workspace of 1 GiB instead.
// A factor that all rows share (1 / count, the gradient of a scalar loss) multiplies the sums, not dz: the label's element
// of dz is near -1 for every row that is not learned yet, and -1 is exact in bf16 where -1/count is off by up to 2^-8 in
// the same direction in every row.
// Bound by the matrix cores.  Logits, statistics, loss and the column sums db are fp32; dz is rounded to the operands'
// type (bf16: half a step 2^-8 of each element, the same rounding that any bf16 product of dz has).
//
// Kernels: the 8-wave 256x256 GEMM (gemm_pingpong.h) for bf16 where its blocks fill the chip, the 4-wave 128x128 one
// (gemm_tiled.h) otherwise and for fp32; logits of few rows or columns by a kernel that shares K between the waves.  Widths that are no multiple of 16 bytes, unaligned or strided operands go through
// zero-padded copies, piece by piece.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gemm_pingpong.h"
#include "gemm_tiled.h"
#include "token_ops.h"

#define DTF_ROR16(v, n) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), 0x120 + (n), 0xf, 0xf, false))

namespace {
enum { VX_LSE = EPI_CUSTOM, VX_DZ = EPI_CUSTOM + 1, VX_SUM = EPI_CUSTOM + 2 };
constexpr int kStrip = 64;                       // columns a wave reduces in the forward pass
constexpr int kLseSplits = 16;                   // waves of the join that share a row's strips

__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, DTF_ROR16(v, 8)); v = fmaxf(v, DTF_ROR16(v, 4)); v = fmaxf(v, DTF_ROR16(v, 2)); v = fmaxf(v, DTF_ROR16(v, 1));
  return v;
}
__device__ __forceinline__ float sum16(float v) {
  v += DTF_ROR16(v, 8); v += DTF_ROR16(v, 4); v += DTF_ROR16(v, 2); v += DTF_ROR16(v, 1);
  return v;
}

// f(0) .. f(N - 1) with compile-time indices: accumulators that are indexed in a loop the compiler leaves rolled (one with
// cross-lane operations under a branch) would live in scratch memory.
template <int I, int N, class F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<I + 1, N>(f);
  }
}

// What the backward pass needs of a row; rows past the last have g = 0.
struct VxRow {
  float lse, g;
  int label, pad;                                // label: -1 where the row has none
};

struct VxGemm : DtfGemmArgs {
  // VX_LSE
  const long long* labels;
  float2* part;                                  // [strips][M]
  float2* target;                                // [M]: the label's logit, whether an earlier column of its strip reaches it
  int v0;                                        // vocabulary index of column 0
  // VX_DZ (C = dz [M, ldc], Ct = dz^T [N, ldct]; both leading dimensions are the padded widths, padding is zeroed)
  const VxRow* rows;                             // padded to the block height
  float* db_part;                                // [wave rows][N], optional
  // VX_SUM: fp32 result C32 [splits][M, ldc32] (accumulate: added to what is there), times *scale if given; with C the
  // sum goes there as bf16 [M, ldc] instead
  const float* scale;
  int kper, accumulate;

  __device__ __forceinline__ void select(int y) {
    if (kper > 0) {
      const int k0 = y * kper;
      const unsigned off = (unsigned)k0 * (dtype == 1 ? 2u : 4u);
      A = static_cast<const char*>(A) + off;
      B = static_cast<const char*>(B) + off;
      a_bytes -= off;
      b_bytes -= off;
      K = min(kper, K - k0);
      C32 += (size_t)y * M * ldc32;
    }
  }

  // acc[ri][cj][r] = C[crow + 16 ri + 4 (lane >> 4) + r][ccol + 16 cj + (lane & 15)]; wl: 16 KB of LDS of this wave
  template <int EPI, int RI>
  __device__ __forceinline__ void epilogue(f32x4 (&acc)[RI][4], unsigned char* wl, int crow, int ccol, int lane) const {
    if (ccol >= N) return;                       // wave-uniform: no column of this block exists
    const int fr = lane & 15, g = lane >> 4;
    if constexpr (EPI == VX_SUM) {
      store_sum<RI>(acc, wl, crow, ccol, lane);
      return;
    }
    const float NEG_INF = -__builtin_huge_valf();
#pragma unroll
    for (int cj = 0; cj < 4; ++cj) {
      const int col = ccol + 16 * cj + fr;
      const float b = bias && col < N ? bias[col] : 0.f;
#pragma unroll
      for (int ri = 0; ri < RI; ++ri)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[ri][cj][r] = col < N ? acc[ri][cj][r] + b : NEG_INF;
    }
    if constexpr (EPI == VX_LSE) {
      float2* const out = part + (size_t)((v0 + ccol) / kStrip) * M;
      bool any = false;
      int off[RI];                               // where in the strip the label of this lane's row lies, or -1
      unrolled<0, RI>([&](auto RIc) {
        constexpr int ri = RIc;
        float om = 0.f, os = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float m = max16(fmaxf(fmaxf(acc[ri][0][r], acc[ri][1][r]), fmaxf(acc[ri][2][r], acc[ri][3][r])));
          const float ref = m == NEG_INF ? 0.f : m;            // a strip masked by its bias: sum 0, not NaN
          const float s = sum16((__expf(acc[ri][0][r] - ref) + __expf(acc[ri][1][r] - ref)) + (__expf(acc[ri][2][r] - ref) + __expf(acc[ri][3][r] - ref)));
          om = fr == r ? m : om;
          os = fr == r ? s : os;
        }
        const int row = crow + 16 * ri + 4 * g + fr;
        const bool mine = fr < 4 && row < M;
        if (mine) out[row] = make_float2(om, os);
        const long long at = mine ? labels[row] - v0 - ccol : -1;
        off[ri] = at >= 0 && at < kStrip && ccol + at < N ? (int)at : -1;
        any |= off[ri] >= 0;
      });
      if (__ballot(any) == 0) return;            // a row's label falls into one strip of V / 64
      unrolled<0, RI>([&](auto RIc) {
        constexpr int ri = RIc;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int o = __shfl(off[ri], (lane & 48) | r);
          // all four shuffled, then chosen: a choice between accumulators would become an indexed load from scratch
          const int from = (lane & 48) | (o & 15), cj = (o >> 4) & 3;
          const float z0 = __shfl(acc[ri][0][r], from), z1 = __shfl(acc[ri][1][r], from), z2 = __shfl(acc[ri][2][r], from), z3 = __shfl(acc[ri][3][r], from);
          const float zt = cj == 0 ? z0 : cj == 1 ? z1 : cj == 2 ? z2 : z3;
          bool earlier = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) earlier |= 16 * k + fr < o && acc[ri][k][r] >= zt;
          const bool dup = (__ballot(earlier) >> (lane & 48)) & 0xffffull;
          if (o >= 0 && fr == 0) target[crow + 16 * ri + 4 * g + r] = make_float2(zt, dup ? 1.f : 0.f);
        }
      });
    } else {
      float db[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ri = 0; ri < RI; ++ri)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const VxRow row = rows[crow + 16 * ri + 4 * g + r];
          const int lab = row.label - v0 - ccol - fr;
#pragma unroll
          for (int cj = 0; cj < 4; ++cj) {
            const float p = __expf(acc[ri][cj][r] - row.lse) - (row.label >= 0 && lab == 16 * cj ? 1.f : 0.f);
            const float v = row.g == 0.f || ccol + 16 * cj + fr >= N ? 0.f : p * row.g;
            acc[ri][cj][r] = v;
            db[cj] += v;
          }
        }
      if (db_part) {
#pragma unroll
        for (int cj = 0; cj < 4; ++cj) {
          float v = db[cj];
          v += __shfl_xor(v, 16);
          v += __shfl_xor(v, 32);
          const int col = ccol + 16 * cj + fr;
          if (g == 0 && col < N) db_part[(size_t)(crow / (16 * RI)) * N + col] = v;
        }
      }
      if (dtype == 1) store_dz16<RI>(acc, wl, crow, ccol, lane);
      else store_dz32<RI>(acc, crow, ccol, lane);
    }
  }

  // fp32: straight from the result layout (a lane holds four rows of a column)
  template <int RI>
  __device__ __forceinline__ void store_dz32(const f32x4 (&acc)[RI][4], int crow, int ccol, int lane) const {
    const int fr = lane & 15, g = lane >> 4;
    float* const c = static_cast<float*>(C);
    float* const ct = static_cast<float*>(Ct);
#pragma unroll
    for (int ri = 0; ri < RI; ++ri)
#pragma unroll
      for (int cj = 0; cj < 4; ++cj) {
        const int row = crow + 16 * ri + 4 * g, col = ccol + 16 * cj + fr;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row + r < M && col < ldc) c[(size_t)(row + r) * ldc + col] = acc[ri][cj][r];
        if (col < N && row < ldct) *reinterpret_cast<f32x4*>(&ct[(size_t)col * ldct + row]) = acc[ri][cj];   // ldct is a multiple of 4
      }
  }

  // bf16: both images are turned in LDS, so that every global store is 16 bytes a lane
  template <int RI>
  __device__ __forceinline__ void store_dz16(const f32x4 (&acc)[RI][4], unsigned char* wl, int crow, int ccol, int lane) const {
    constexpr int CH = 2 * RI;                   // 16-byte chunks of a transposed row (16 RI rows of dz)
    const int fr = lane & 15, g = lane >> 4;
    unsigned short* const c = static_cast<unsigned short*>(C);
    unsigned short* const ct = static_cast<unsigned short*>(Ct);
    uint2 pk[RI][4];
#pragma unroll
    for (int ri = 0; ri < RI; ++ri)
#pragma unroll
      for (int cj = 0; cj < 4; ++cj) {
        pk[ri][cj].x = tk_pack2(acc[ri][cj][0], acc[ri][cj][1]);
        pk[ri][cj].y = tk_pack2(acc[ri][cj][2], acc[ri][cj][3]);
      }
#pragma unroll
    for (int ri = 0; ri < RI; ++ri)
#pragma unroll
      for (int cj = 0; cj < 4; ++cj) {
        const int col = 16 * cj + fr, q = 2 * ri + (g >> 1);
        *reinterpret_cast<uint2*>(&wl[col * CH * 16 + ((q ^ (col & (CH - 1))) << 4) + 8 * (g & 1)]) = pk[ri][cj];
      }
#pragma unroll
    for (int it = 0; it < CH; ++it) {
      const int col = it * (64 / CH) + lane / CH, q = lane & (CH - 1);
      const u32x4 v = *reinterpret_cast<const u32x4*>(&wl[col * CH * 16 + ((q ^ (col & (CH - 1))) << 4)]);
      if (ccol + col < N && crow + q * 8 < ldct) *reinterpret_cast<u32x4*>(&ct[(size_t)(ccol + col) * ldct + crow + q * 8]) = v;
    }
#pragma unroll
    for (int ri = 0; ri < RI; ++ri)
#pragma unroll
      for (int cj = 0; cj < 4; ++cj)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int R = 16 * ri + 4 * g + r, col = 16 * cj + fr;
          const unsigned w32 = r < 2 ? pk[ri][cj].x : pk[ri][cj].y;
          *reinterpret_cast<unsigned short*>(&wl[R * 128 + ((((col >> 3) ^ (R >> 2)) & 7) << 4) + (col & 7) * 2]) = (unsigned short)((r & 1) ? (w32 >> 16) : (w32 & 0xffff));
        }
#pragma unroll
    for (int it = 0; it < 2 * RI; ++it) {
      const int R = it * 8 + (lane >> 3), q = lane & 7;
      const u32x4 v = *reinterpret_cast<const u32x4*>(&wl[R * 128 + (((q ^ (R >> 2)) & 7) << 4)]);
      if (crow + R < M && ccol + q * 8 < ldc) *reinterpret_cast<u32x4*>(&c[(size_t)(crow + R) * ldc + ccol + q * 8]) = v;
    }
  }

  // 64 rows at a time through LDS as fp32; N (a padded width) and the leading dimensions are multiples of 4
  template <int RI>
  __device__ __forceinline__ void store_sum(const f32x4 (&acc)[RI][4], unsigned char* wl, int crow, int ccol, int lane) const {
    const int fr = lane & 15, g = lane >> 4;
    const float f = scale ? *scale : 1.f;
    unsigned short* const c16 = static_cast<unsigned short*>(C);
#pragma unroll
    for (int h = 0; h < RI / 4; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int cj = 0; cj < 4; ++cj)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int R = 16 * i + 4 * g + r, col = 16 * cj + fr;
            *reinterpret_cast<float*>(&wl[R * 256 + ((((col >> 2) ^ (R >> 2)) & 15) << 4) + (col & 3) * 4]) = acc[4 * h + i][cj][r];
          }
#pragma unroll
      for (int it = 0; it < 16; ++it) {
        const int R = it * 4 + (lane >> 4), q = lane & 15;
        f32x4 v = *reinterpret_cast<const f32x4*>(&wl[R * 256 + (((q ^ (R >> 2)) & 15) << 4)]);
        const int row = crow + 64 * h + R, col = ccol + q * 4;
        if (row < M && col < N) {
          f32x4* const p = reinterpret_cast<f32x4*>(&C32[(size_t)row * ldc32 + col]);
          if (accumulate) {
            const f32x4 o = *p;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += o[e];
          }
          if (scale) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= f;
          }
          if (c16) *reinterpret_cast<uint2*>(&c16[(size_t)row * ldc + col]) = make_uint2(tk_pack2(v[0], v[1]), tk_pack2(v[2], v[3]));
          else *p = v;
        }
      }
    }
  }
};

// Few rows, or few columns: 16 rows x 64 columns a workgroup, the four waves share K (64 bytes of a row a step, wave by
// wave), operands straight from memory into the matrix instructions: one wave's 20 loads in flight, no staging, no barrier
// in the loop.  Every row of W is read by ceil(M / 16) workgroups, next to each other on one XCD.
template <typename T, int EPI>
__global__ __launch_bounds__(256) void vx_skinny_kernel(VxGemm p) {
  constexpr int PER16 = Elem<T>::PER16, AHEAD = 4;
  __shared__ float s_acc[3][16][64];
  __shared__ __attribute__((aligned(16))) unsigned char s_out[2048];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, g = lane >> 4;
  const int tiles_m = (p.M + 15) >> 4, wg = dtf_xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = (wg % tiles_m) * 16, n0 = (wg / tiles_m) * 64;
  const rsrc_t ra = make_rsrc(p.A, p.a_bytes), rb = make_rsrc(p.B, p.b_bytes);
  const unsigned a_off = m0 + fr < p.M ? (unsigned)(m0 + fr) * (unsigned)p.lda * (unsigned)sizeof(T) : kOOB;
  unsigned b_off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b_off[j] = n0 + 16 * j + fr < p.N ? (unsigned)(n0 + 16 * j + fr) * (unsigned)p.ldb * (unsigned)sizeof(T) : kOOB;
  f32x4 acc[1][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (p.K + 4 * PER16 - 1) / (4 * PER16);
  for (int s = wave; s < steps; s += 4 * AHEAD) {
    u32x4 a[AHEAD], b[AHEAD][4];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = (s + 4 * u) * 4 + g;           // 16-byte piece of the row
      const bool in = k * PER16 < p.K;
      a[u] = __builtin_amdgcn_raw_buffer_load_b128(ra, (int)(in && a_off != kOOB ? a_off + k * 16u : kOOB), 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[u][j] = __builtin_amdgcn_raw_buffer_load_b128(rb, (int)(in && b_off[j] != kOOB ? b_off[j] + k * 16u : kOOB), 0, 0);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_slot<T>(a[u], b[u][j], acc[0][j]);
  }
  if (wave) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) s_acc[wave - 1][4 * j + r][lane] = acc[0][j][r];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[0][j][r] = ((acc[0][j][r] + s_acc[0][4 * j + r][lane]) + s_acc[1][4 * j + r][lane]) + s_acc[2][4 * j + r][lane];
  p.template epilogue<EPI>(acc, s_out, m0, n0, lane);
}

// ------------------------------------------------------------------------------------------------- streaming helpers
// dst[r, 0 .. ldd) = src[r, 0 .. cols) and zeros: an aligned, padded copy in the operands' type.
template <typename TS, typename TD>
__global__ __launch_bounds__(256) void vx_pack_kernel(const TS* __restrict__ src, TD* __restrict__ dst, int rows, int cols, long lds_, int ldd) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, row = i / ldd;
  const int c = (int)(i - row * ldd);
  if (row >= rows) return;
  tk_put(dst + i, c < cols ? tk_get(src + row * lds_ + c) : 0.f);
}

// dst[c, r] = src[r, c] for r < M, c < N; zeros for r in [M, ldt).  64 x 64 tiles through LDS.
template <typename T>
__global__ __launch_bounds__(256) void vx_transpose_kernel(const T* __restrict__ src, T* __restrict__ dst, int M, int N, long lds_, int ldt) {
  constexpr int PER16 = 16 / sizeof(T);
  __shared__ T tile[64][64 + PER16];
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
  constexpr int CH = 64 / PER16;               // 16-byte chunks of a tile row
#pragma unroll
  for (int i = 0; i < CH / 4; ++i) {
    const int id = threadIdx.x + 256 * i, rr = id / CH, ch = id % CH;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (r0 + rr < M && c0 + ch * PER16 < N) v = *reinterpret_cast<const u32x4*>(src + (size_t)(r0 + rr) * lds_ + c0 + ch * PER16);
    *reinterpret_cast<u32x4*>(&tile[rr][ch * PER16]) = v;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < CH / 4; ++i) {
    const int id = threadIdx.x + 256 * i, cc = id / CH, ch = id % CH;
    if (c0 + cc >= N || r0 + ch * PER16 >= ldt) continue;
    alignas(16) T e[PER16];
#pragma unroll
    for (int k = 0; k < PER16; ++k) e[k] = tile[ch * PER16 + k][cc];
    *reinterpret_cast<u32x4*>(dst + (size_t)(c0 + cc) * ldt + r0 + ch * PER16) = *reinterpret_cast<u32x4*>(e);
  }
}

// out[r, c] = scale * sum of the splits' fp32 results, in their order, rounded to the output's type.
template <typename T>
__global__ __launch_bounds__(256) void vx_finish_kernel(const float* __restrict__ ws, int splits, int rows, int cols, int ldw, T* __restrict__ out, long ldo,
                                                        const float* __restrict__ scale) {
  const int quads = (cols + 3) >> 2;
  const long i = (long)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  const int c = (int)(i - row * quads) * 4;
  if (row >= rows) return;
  f32x4 v = *reinterpret_cast<const f32x4*>(ws + (size_t)row * ldw + c);
  for (int s = 1; s < splits; ++s) {
    const f32x4 o = *reinterpret_cast<const f32x4*>(ws + ((size_t)s * rows + row) * ldw + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += o[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < cols) tk_put(out + row * ldo + c + e, v[e] * *scale);
}

// db[c] = scale * sum of the wave rows' partial column sums
__global__ __launch_bounds__(256) void vx_db_kernel(const float* __restrict__ part, int nparts, int N, float* __restrict__ db, const float* __restrict__ scale) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float v = 0.f;
  for (int p = 0; p < nparts; ++p) v += part[(size_t)p * N + c];
  db[c] = v * *scale;
}

__global__ __launch_bounds__(256) void vx_rows_kernel(const float* __restrict__ lse, const long long* __restrict__ labels, const float* __restrict__ dloss,
                                                      int dloss_rows, const long long* __restrict__ counts, int mean, int M, int Mp, long V,
                                                      long long ignore, VxRow* __restrict__ rows, float* __restrict__ scale) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r == 0) {
    const float up = dloss && !dloss_rows ? *dloss : 1.f;
    *scale = mean ? (counts[1] ? up / (float)counts[1] : 0.f) : up;
  }
  if (r >= Mp) return;
  VxRow o = {0.f, 0.f, -1, 0};
  if (r < M) {
    const long long lab = labels[r];
    if (lab != ignore && lab >= 0 && lab < V) {
      o.lse = lse[r];
      o.g = dloss_rows ? dloss[r] : 1.f;
      o.label = (int)lab;
    }
  }
  rows[r] = o;
}

// (m, s) += (m2, s2): running maximum and sum of exponentials; -inf with sum 0 is the neutral element.
__device__ __forceinline__ void lse_add(float& m, float& s, float m2, float s2) {
  const float big = fmaxf(m, m2), ref = big == -__builtin_huge_valf() ? 0.f : big;
  s = s * __expf(m - ref) + s2 * __expf(m2 - ref);
  m = big;
}

// 64 rows a workgroup, 16 waves share a row's strips.  block_out: this workgroup's sums, or (last = only workgroup) the result.
struct VxJoin {
  const float2* part; const float2* target; const long long* labels;
  float* lse; float* loss_rows; float* loss; long long* counts; float* blk_loss; int* blk_counts;
  int M, strips, blocks, mean; long V; long long ignore;
};

__device__ __forceinline__ void vx_result(const VxJoin& a, float loss, long long hits, long long n) {
  *a.loss = a.mean ? (n ? loss / (float)n : 0.f) : loss;
  a.counts[0] = hits;
  a.counts[1] = n;
}

__global__ __launch_bounds__(64 * kLseSplits) void vx_join_kernel(VxJoin a) {
  __shared__ float s_m[kLseSplits][64], s_s[kLseSplits][64];
  __shared__ int s_first[kLseSplits][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x * 64 + lane;
  float m = -__builtin_huge_valf(), s = 0.f;
  int first = 0x7fffffff;                        // the first strip that reaches the maximum
  if (row < a.M)
    for (int k = wave; k < a.strips; k += 4 * kLseSplits) {
      float2 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        p[u] = k + u * kLseSplits < a.strips ? a.part[(size_t)(k + u * kLseSplits) * a.M + row] : make_float2(-__builtin_huge_valf(), 0.f);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (p[u].x > m) first = k + u * kLseSplits;
        lse_add(m, s, p[u].x, p[u].y);
      }
    }
  s_m[wave][lane] = m;
  s_s[wave][lane] = s;
  s_first[wave][lane] = first;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kLseSplits; ++w) {
    const float m2 = s_m[w][lane];
    const int f2 = s_first[w][lane];
    if (m2 > m || (m2 == m && f2 < first)) first = f2;
    lse_add(m, s, m2, s_s[w][lane]);
  }
  float loss = 0.f;
  int hit = 0, valid = 0;
  if (row < a.M) {
    const float lse = m + logf(s);
    const long long lab = a.labels[row];
    a.lse[row] = lse;
    if (lab != a.ignore) {
      valid = 1;
      if (lab >= 0 && lab < a.V) {
        const float2 t = a.target[row];
        loss = lse - t.x;
        hit = t.x >= m && first == (int)(lab / kStrip) && t.y == 0.f;
      } else {
        loss = __builtin_nanf("");               // no such class
      }
    }
    a.loss_rows[row] = loss;
  }
  loss = tk_wave_sum(loss);
  const int hits = (int)__popcll(__ballot(hit)), n = (int)__popcll(__ballot(valid));
  if (lane == 0) {
    if (a.blocks == 1) vx_result(a, loss, hits, n);
    else {
      a.blk_loss[blockIdx.x] = loss;
      a.blk_counts[2 * blockIdx.x] = hits;
      a.blk_counts[2 * blockIdx.x + 1] = n;
    }
  }
}

__global__ __launch_bounds__(256) void vx_total_kernel(VxJoin a) {
  __shared__ float s_l[4];
  __shared__ int s_h[4], s_n[4];
  float loss = 0.f;
  int hits = 0, n = 0;                           // at most M
  for (int b = threadIdx.x; b < a.blocks; b += 256) {
    loss += a.blk_loss[b];
    hits += a.blk_counts[2 * b];
    n += a.blk_counts[2 * b + 1];
  }
  loss = tk_wave_sum(loss);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { hits += __shfl_xor(hits, d); n += __shfl_xor(n, d); }
  if ((threadIdx.x & 63) == 0) { s_l[threadIdx.x >> 6] = loss; s_h[threadIdx.x >> 6] = hits; s_n[threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x == 0) vx_result(a, (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]), s_h[0] + s_h[1] + s_h[2] + s_h[3], s_n[0] + s_n[1] + s_n[2] + s_n[3]);
}

// --------------------------------------------------------------------------------------------------------- host side
long up(long v, long to) { return (v + to - 1) / to * to; }

// 256x256 blocks of the 8-wave kernel where they fill the chip (its staging offsets ask for whole half-tiles in range)
bool use_pp(int dtype, long m, long n, long k, int splits) {
  return dtype == TK_BF16 && m >= 256 && n >= 256 && k / splits >= 256 && ((m + 255) / 256) * ((n + 255) / 256) * splits >= 192;
}

// 128x128 blocks would leave most CUs idle, or their rows mostly empty
bool use_skinny(long m, long n) { return m <= 16 || ((m + 127) / 128) * ((n + 127) / 128) < 128; }

// Rows of a wave's block in the logits' epilogue
int wave_rows(const VxGemm& a) { return use_skinny(a.M, a.N) ? 16 : use_pp(a.dtype, a.M, a.N, a.K, 1) ? 128 : 64; }

template <int EPI>
void launch_gemm(const VxGemm& a, int splits, hipStream_t s) {
  if (use_pp(a.dtype, a.M, a.N, a.K, splits)) {
    const dim3 g(dtf_cdiv(a.M, 256) * dtf_cdiv(a.N, 256), splits);
    hipLaunchKernelGGL((gemm_pp_kernel<EPI, VxGemm>), g, dim3(512), 0, s, a);
  } else {
    const dim3 g(dtf_cdiv(a.M, 128) * dtf_cdiv(a.N, 128), splits);
    if (a.dtype == TK_BF16) hipLaunchKernelGGL((gemm_tiled_kernel<unsigned short, EPI, 4, 4, VxGemm>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((gemm_tiled_kernel<unsigned int, EPI, 4, 4, VxGemm>), g, dim3(256), 0, s, a);
  }
}

template <int EPI>
void launch_logits(const VxGemm& a, hipStream_t s) {
  if (!use_skinny(a.M, a.N)) return launch_gemm<EPI>(a, 1, s);
  const dim3 g((unsigned)(dtf_cdiv(a.M, 16) * dtf_cdiv(a.N, 64)));
  if (a.dtype == TK_BF16) hipLaunchKernelGGL((vx_skinny_kernel<unsigned short, EPI>), g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((vx_skinny_kernel<unsigned int, EPI>), g, dim3(256), 0, s, a);
}

VxGemm operands(const void* A, const void* B, int dtype, int M, int N, int K, long lda, long ldb) {
  VxGemm g = {};
  const long es = dtype == TK_BF16 ? 2 : 4;
  g.A = A; g.B = B; g.M = M; g.N = N; g.K = K;
  g.lda = (int)lda; g.ldb = (int)ldb; g.dtype = dtype;
  g.a_bytes = (unsigned)(((M - 1) * lda + K) * es);
  g.b_bytes = (unsigned)(((N - 1) * ldb + K) * es);
  return g;
}

// How many K ranges a product is cut into, so that its blocks fill the chip: 256x256 blocks (one a CU) if they do with
// ranges of 1024 or more, else 128x128 blocks (two a CU), at least 512 deep.
int splits_for(int dtype, long m, long n, long k) {
  if (dtype == TK_BF16 && m >= 256 && n >= 256) {
    const long big = ((m + 255) / 256) * ((n + 255) / 256), s = std::max<long>(1, 256 / big);
    if (big * s >= 192 && k / s >= 1024) return (int)s;
  }
  const long blocks = ((m + 127) / 128) * ((n + 127) / 128);
  return (int)std::max<long>(1, std::min<long>({512 / blocks, k / 512, 32}));
}
long kper_for(long k, int splits) { return up((k + splits - 1) / splits, 128); }

// Sizes of one call: the padded width, the vocabulary piece and the workspace's parts
struct VxPlan {
  long es, per16, Dp, Np, Vp, pieces, strips, blocks;
  bool pack_x, pack_w, direct_dx, direct_dw;
  int sx, sw;                                    // splits of the two products
  size_t x, w, part, target, blk, rows, xt, wt, dz, dzt, dx32, dw32, db, total;
};

size_t take(size_t& at, size_t bytes) {
  const size_t here = at;
  at += (bytes + 255) & ~(size_t)255;
  return here;
}

VxPlan plan(const DtfVocabXentArgs& a, bool backward) {
  VxPlan p = {};
  p.es = a.dtype == TK_BF16 ? 2 : 4;
  p.per16 = 16 / p.es;
  p.Dp = up(a.D, p.per16);
  p.Np = up(a.N, 8);
  p.pack_x = a.D % p.per16 || a.ldx % p.per16 || !dtf_aligned16(a.X);
  p.pack_w = a.w_dtype != a.dtype || a.D % p.per16 || a.ldw % p.per16 || !dtf_aligned16(a.W);
  // a piece: dz and its transpose in 1 GiB, but never under 16384 columns (the products' K and M); every operand of a
  // launch stays below 2 GiB (32-bit offsets)
  long vp = backward ? std::max<long>((1l << 30) / (2 * p.es * p.Np), 16384) : (1l << 30);
  vp = std::min(vp, ((1l << 31) - (1 << 20)) / (p.es * std::max(p.Dp, backward ? p.Np : 0)));
  vp = std::max<long>(vp / 256 * 256, 256);
  p.pieces = (a.V + vp - 1) / vp;
  p.Vp = p.pieces == 1 ? a.V : std::min(vp, up((a.V + p.pieces - 1) / p.pieces, 256));
  p.pieces = (a.V + p.Vp - 1) / p.Vp;
  size_t at = 0;
  if (p.pack_x) p.x = take(at, (size_t)a.N * p.Dp * p.es);
  if (p.pack_w) p.w = take(at, (size_t)p.Vp * p.Dp * p.es);
  if (!backward) {
    p.strips = (a.V + kStrip - 1) / kStrip;
    p.blocks = (a.N + 63) / 64;
    p.part = take(at, (size_t)p.strips * a.N * 8);
    p.target = take(at, (size_t)a.N * 8);
    p.blk = take(at, (size_t)p.blocks * 12);
  } else {
    const long Vpp = up(p.Vp, 8);
    p.rows = take(at, (size_t)up(a.N, 256) * sizeof(VxRow) + 16);     // and the common factor behind them
    p.xt = take(at, (size_t)p.Dp * p.Np * p.es);
    p.wt = take(at, (size_t)p.Dp * Vpp * p.es);
    p.dz = take(at, (size_t)a.N * Vpp * p.es);
    p.dzt = take(at, (size_t)p.Vp * p.Np * p.es);
    p.sx = splits_for(a.dtype, a.N, p.Dp, Vpp);
    p.sw = splits_for(a.dtype, p.Vp, p.Dp, p.Np);
    p.sx = (int)((Vpp + kper_for(Vpp, p.sx) - 1) / kper_for(Vpp, p.sx));
    p.sw = (int)((p.Np + kper_for(p.Np, p.sw) - 1) / kper_for(p.Np, p.sw));
    // straight into the result where one product (or the last piece's) holds the whole sum at a 16-byte row width
    p.direct_dx = p.sx == 1 && p.Dp == a.D && dtf_aligned16(a.dX);
    p.direct_dw = p.sw == 1 && p.Dp == a.D && dtf_aligned16(a.dW);
    if (!p.direct_dx || (a.dtype == TK_BF16 && p.pieces > 1)) p.dx32 = take(at, (size_t)p.sx * a.N * p.Dp * 4);
    if (!p.direct_dw) p.dw32 = take(at, (size_t)p.sw * p.Vp * p.Dp * 4);
    if (a.dbias) p.db = take(at, (size_t)(a.N / 16 + 4) * p.Vp * 4);       // one row of partial sums for every 16 rows at most
  }
  p.total = at;
  return p;
}

template <typename T>
void finish_as(const float* ws, int splits, long rows, int cols, int ldw, void* out, long ldo, const float* scale, hipStream_t s) {
  const long n = rows * ((cols + 3) / 4);
  hipLaunchKernelGGL((vx_finish_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, ws, splits, (int)rows, cols, ldw, static_cast<T*>(out), ldo, scale);
}
void finish(const float* ws, int splits, long rows, int cols, int ldw, void* out, long ldo, int dtype, const float* scale, hipStream_t s) {
  if (dtype == TK_BF16) finish_as<unsigned short>(ws, splits, rows, cols, ldw, out, ldo, scale, s);
  else finish_as<float>(ws, splits, rows, cols, ldw, out, ldo, scale, s);
}

template <typename TS, typename TD>
void pack_as(const void* src, void* dst, long rows, int cols, long lds_, long ldd, hipStream_t s) {
  hipLaunchKernelGGL((vx_pack_kernel<TS, TD>), dim3((unsigned)((rows * ldd + 255) / 256)), dim3(256), 0, s, static_cast<const TS*>(src),
                     static_cast<TD*>(dst), (int)rows, cols, lds_, (int)ldd);
}
void pack(const void* src, int sdt, void* dst, int ddt, long rows, int cols, long lds_, long ldd, hipStream_t s) {
  if (ddt == TK_F32) pack_as<float, float>(src, dst, rows, cols, lds_, ldd, s);
  else if (sdt == TK_F32) pack_as<float, unsigned short>(src, dst, rows, cols, lds_, ldd, s);
  else pack_as<unsigned short, unsigned short>(src, dst, rows, cols, lds_, ldd, s);
}

void transpose(const void* src, void* dst, long M, long N, long lds_, long ldt, int dtype, hipStream_t s) {
  const dim3 g((unsigned)((N + 63) / 64), (unsigned)((ldt + 63) / 64));
  if (dtype == TK_BF16)
    hipLaunchKernelGGL((vx_transpose_kernel<unsigned short>), g, dim3(256), 0, s, static_cast<const unsigned short*>(src), static_cast<unsigned short*>(dst), (int)M, (int)N, lds_, (int)ldt);
  else
    hipLaunchKernelGGL((vx_transpose_kernel<float>), g, dim3(256), 0, s, static_cast<const float*>(src), static_cast<float*>(dst), (int)M, (int)N, lds_, (int)ldt);
}

int check(const DtfVocabXentArgs* a) {
  if (!a) return DTF_ERR_ARG;
  if ((a->dtype != TK_F32 && a->dtype != TK_BF16) || (a->w_dtype != TK_F32 && a->w_dtype != TK_BF16)) return DTF_ERR_ARG;
  if (a->w_dtype == TK_BF16 && a->dtype == TK_F32) return DTF_ERR_ARG;
  if (a->N <= 0 || a->V <= 0 || a->D <= 0 || a->ldx < a->D || a->ldw < a->D) return DTF_ERR_SHAPE;
  const long es = a->dtype == TK_BF16 ? 2 : 4, limit = (1l << 31) - (1 << 20);
  if (a->V > (1l << 30) || a->N > (1l << 26) || a->D > (1l << 20)) return DTF_ERR_SHAPE;
  if ((long)a->N * std::max<long>(a->ldx, up(a->D, 8)) * es > limit || (long)up(a->D, 8) * 256 * es > limit || (long)up(a->N, 8) * 256 * es > limit) return DTF_ERR_SHAPE;
  if (a->ldw > limit / (256 * es)) return DTF_ERR_SHAPE;
  return DTF_OK;
}
}  // namespace

DTF_EXPORT int64_t dtf_vocab_xent_ws_bytes(const DtfVocabXentArgs* a, int backward) {
  return check(a) == DTF_OK ? (int64_t)plan(*a, backward != 0).total : -1;
}

DTF_EXPORT int dtf_vocab_xent_fwd(const DtfVocabXentArgs* ap, hipStream_t s) {
  if (const int rc = check(ap)) return rc;
  const DtfVocabXentArgs& a = *ap;
  if (!a.X || !a.W || !a.labels || !a.lse || !a.loss_rows || !a.loss || !a.counts || !a.ws) return DTF_ERR_ARG;
  const VxPlan p = plan(a, false);
  if (a.ws_bytes < (int64_t)p.total) return DTF_ERR_SHAPE;
  if (!dtf_aligned16(a.ws)) return DTF_ERR_ALIGN;
  char* const ws = static_cast<char*>(a.ws);
  const void* X = a.X;
  long ldx = a.ldx;
  if (p.pack_x) {
    pack(a.X, a.dtype, ws + p.x, a.dtype, a.N, a.D, a.ldx, p.Dp, s);
    X = ws + p.x;
    ldx = p.Dp;
  }
  for (long v0 = 0; v0 < a.V; v0 += p.Vp) {
    const long n = std::min<long>(p.Vp, a.V - v0);
    const void* W = static_cast<const char*>(a.W) + v0 * a.ldw * (a.w_dtype == TK_BF16 ? 2 : 4);
    long ldw = a.ldw;
    if (p.pack_w) {
      pack(W, a.w_dtype, ws + p.w, a.dtype, n, a.D, a.ldw, p.Dp, s);
      W = ws + p.w;
      ldw = p.Dp;
    }
    VxGemm g = operands(X, W, a.dtype, a.N, (int)n, (int)p.Dp, ldx, ldw);
    g.bias = a.bias ? a.bias + v0 : nullptr;
    g.labels = a.labels;
    g.part = reinterpret_cast<float2*>(ws + p.part);
    g.target = reinterpret_cast<float2*>(ws + p.target);
    g.v0 = (int)v0;
    launch_logits<VX_LSE>(g, s);
  }
  VxJoin j = {reinterpret_cast<const float2*>(ws + p.part), reinterpret_cast<const float2*>(ws + p.target), a.labels, a.lse, a.loss_rows, a.loss,
              a.counts, reinterpret_cast<float*>(ws + p.blk), reinterpret_cast<int*>(ws + p.blk + p.blocks * 4), a.N, (int)p.strips, (int)p.blocks,
              a.mean, a.V, a.ignore};
  hipLaunchKernelGGL(vx_join_kernel, dim3((unsigned)p.blocks), dim3(64 * kLseSplits), 0, s, j);
  if (p.blocks > 1) hipLaunchKernelGGL(vx_total_kernel, dim3(1), dim3(256), 0, s, j);
  return dtf_check_launch();
}

DTF_EXPORT int dtf_vocab_xent_bwd(const DtfVocabXentArgs* ap, hipStream_t s) {
  if (const int rc = check(ap)) return rc;
  const DtfVocabXentArgs& a = *ap;
  if (!a.X || !a.W || !a.labels || !a.lse || !a.counts || !a.ws || !(a.dX || a.dW || a.dbias)) return DTF_ERR_ARG;
  const VxPlan p = plan(a, true);
  if (a.ws_bytes < (int64_t)p.total) return DTF_ERR_SHAPE;
  if (!dtf_aligned16(a.ws)) return DTF_ERR_ALIGN;
  char* const ws = static_cast<char*>(a.ws);
  const void* X = a.X;
  long ldx = a.ldx;
  if (p.pack_x) {
    pack(a.X, a.dtype, ws + p.x, a.dtype, a.N, a.D, a.ldx, p.Dp, s);
    X = ws + p.x;
    ldx = p.Dp;
  }
  VxRow* const rows = reinterpret_cast<VxRow*>(ws + p.rows);
  const int Mp = (int)up(a.N, 256);
  float* const scale = reinterpret_cast<float*>(rows + Mp);
  hipLaunchKernelGGL(vx_rows_kernel, dim3(Mp / 256), dim3(256), 0, s, a.lse, a.labels, a.dloss, a.dloss_rows, a.counts, a.mean, a.N, Mp, a.V, a.ignore, rows, scale);
  if (a.dW) transpose(X, ws + p.xt, a.N, p.Dp, ldx, p.Np, a.dtype, s);
  float* const dx32 = reinterpret_cast<float*>(ws + p.dx32);
  float* const dw32 = reinterpret_cast<float*>(ws + p.dw32);
  for (long v0 = 0; v0 < a.V; v0 += p.Vp) {
    const long n = std::min<long>(p.Vp, a.V - v0), np = up(n, 8);
    const void* W = static_cast<const char*>(a.W) + v0 * a.ldw * (a.w_dtype == TK_BF16 ? 2 : 4);
    long ldw = a.ldw;
    if (p.pack_w) {
      pack(W, a.w_dtype, ws + p.w, a.dtype, n, a.D, a.ldw, p.Dp, s);
      W = ws + p.w;
      ldw = p.Dp;
    }
    VxGemm g = operands(X, W, a.dtype, a.N, (int)n, (int)p.Dp, ldx, ldw);
    g.bias = a.bias ? a.bias + v0 : nullptr;
    g.rows = rows;
    g.v0 = (int)v0;
    g.C = ws + p.dz;
    g.ldc = (int)np;
    g.Ct = ws + p.dzt;
    g.ldct = (int)p.Np;
    g.db_part = a.dbias ? reinterpret_cast<float*>(ws + p.db) : nullptr;
    launch_logits<VX_DZ>(g, s);
    if (a.dbias) {
      hipLaunchKernelGGL(vx_db_kernel, dim3(dtf_cdiv((int)n, 256)), dim3(256), 0, s, g.db_part, dtf_cdiv(a.N, wave_rows(g)), (int)n, a.dbias + v0, scale);
    }
    if (a.dX) {
      transpose(W, ws + p.wt, n, p.Dp, ldw, np, a.dtype, s);
      VxGemm d = operands(ws + p.dz, ws + p.wt, a.dtype, a.N, (int)p.Dp, (int)np, np, np);
      const long kper = kper_for(up(p.Vp, 8), p.sx);
      const int splits = (int)((np + kper - 1) / kper);
      d.kper = p.sx > 1 ? (int)kper : 0;
      d.C32 = p.direct_dx && a.dtype == TK_F32 ? static_cast<float*>(a.dX) : dx32;
      d.ldc32 = (int)p.Dp;
      d.accumulate = v0 > 0;                     // the last, shorter piece adds to its first splits only
      if (p.direct_dx && v0 + n == a.V) {
        d.scale = scale;
        if (a.dtype == TK_BF16) d.C = a.dX;
        d.ldc = a.D;
      }
      launch_gemm<VX_SUM>(d, splits, s);
    }
    if (a.dW) {
      VxGemm d = operands(ws + p.dzt, ws + p.xt, a.dtype, (int)n, (int)p.Dp, (int)p.Np, p.Np, p.Np);
      d.kper = p.sw > 1 ? (int)kper_for(p.Np, p.sw) : 0;
      void* const out = static_cast<char*>(a.dW) + v0 * a.D * (a.w_dtype == TK_BF16 ? 2 : 4);
      d.C32 = p.direct_dw && a.w_dtype == TK_F32 ? static_cast<float*>(out) : dw32;
      d.ldc32 = (int)p.Dp;
      if (p.direct_dw) {
        d.scale = scale;
        if (a.w_dtype == TK_BF16) d.C = out;
        d.ldc = a.D;
      }
      launch_gemm<VX_SUM>(d, p.sw, s);
      if (!p.direct_dw) finish(dw32, p.sw, n, a.D, (int)p.Dp, out, a.D, a.w_dtype, scale, s);
    }
  }
  if (a.dX && !p.direct_dx) finish(dx32, p.sx, a.N, a.D, (int)p.Dp, a.dX, a.D, a.dtype, scale, s);
  return dtf_check_launch();
}
