// Softmax cross entropy over a large vocabulary without keeping the logits: z = X W^T + b, X [N tokens, D], W [V, D].
//
//   forward    lse_r = log sum_c exp z_rc;   loss_r = lse_r - z_r,label;   hit_r: label is the first maximum of the row
//   backward   dz_rc = (exp z_rc / sum_c exp z_rc - [c = label_r]) g_r;   dX = dz W;   dW = dz^T X;   db_c = sum_r dz_rc
//
// Forward: one GEMM whose epilogue reduces each row of a wave's 64-column strip to (maximum, sum of exponentials) and
// picks the label's logit on the way; a join over the strips gives lse, loss and hits.  8 bytes a strip and row leave the
// chip instead of 256 of logits.
// Backward: the vocabulary is cut into pieces; for each piece the same GEMM is run again and its epilogue writes dz in the
// operands' type, once as [N, piece] and once transposed, which are the operands of the two products dX += dz W and
// dW = dz^T X (all products in the one form A[M,K] . B[N,K]^T of the tiled GEMMs).  The work is 8 N V D operations instead
// of the 6 N V D of a program that stores the logits: at N = 8192, V = 131072 the fp32 logits would be 4 GB to write and
// read again, 2.1 GB of bf16 dz per step go through a workspace of 1 GiB instead.
// What multiplies a whole row of dz (1 / count, the gradient of a scalar loss or of the row's own) stays out of dz where dz is
// rounded to bf16: the label's element of dz is near -1 for every row that is not learned yet, and -1 is exact in bf16
// where -1/count is off by up to 2^-8 in the same direction in every row.  The factor that the rows share multiplies the
// sums (of gradients a row: the largest of them); what is left of a row's own, 1 where all are equal, multiplies its row of dX,
// its share of db, and its X in the transposed copy that dW reads.
// Bound by the matrix cores, which the products keep 74-86 % busy: 8192 x 131072 x 4096 bf16 takes 25.1 ms forward and
// backward, 1400 TFLOP/s over the 8 N V D (a large library product: 1350); 4093 x 50001 x 1024 1.6 ms, where the epilogues of
// the logits' launches are a third of their time; 777 x 10007 x 512 fp32 0.36 ms.  Few rows are bound by reading W (bf16, 16
// rows at 65536 x 4096 forward and backward 0.56 ms: four passes over 0.54 GB), in fp32 from some 40 rows on by cutting and
// multiplying planes (64 rows 1.24 ms: 111 TFLOP/s over the 8 N V D, a large fp32 library product 155).
// Logits, statistics, loss and the column sums db are fp32; dz is rounded to the operands' type (bf16: half a step 2^-8 of
// each element, the same rounding that any bf16 product of dz has).
//
// fp32 operands are cut into three bf16 planes, x = x0 + x1 + x2 up to 2^-26 |x| (each plane takes eight more bits), and a
// product is the sum of the six plane products x0 w0, x0 w1, x1 w0, x0 w2, x2 w0, x1 w1, accumulated in fp32; what is left out
// is below 2^-25 of |x w|, under an fp32 rounding.  Six bf16 matrix products cost less than one in fp32, whose matrix rate is
// a sixteenth.  (Elements below 2^-110 lose their last planes: 10^-33 beside sums of order one.)  An infinity has no planes
// that a sum of six products could be made of (0 or a remainder of the other sign times infinity is NaN), and a finite
// number may round to one in its first plane: whoever finds infinities or NaN in its sums makes them again from the
// operands as they are, with fp32 instructions, and takes those that were not finite from there (the others keep their
// bits: what a neighbouring row holds does not matter).  Finite operands pay one instruction for every element of the result.
// The large products dX and dW of planes cut beforehand do not: an infinity that meets a dz other than 0 (its row's loss is
// infinite then) gives NaN.
//
// Kernels: the 8-wave 256x256 GEMM (gemm_pingpong.h) where its blocks fill the chip, the 4-wave 128x128 one (gemm_tiled.h)
// otherwise; logits of few rows or columns by kernels that share K between the waves; the products of few rows by kernels that
// read W and write dW once, with fp32 matrix instructions or, fp32 operands of 17 rows and more, planes cut in registers.
// bf16 widths that are no multiple of 16 bytes, unaligned or strided operands go through zero-padded copies, piece by piece.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gemm_pingpong.h"
#include "gemm_tiled.h"
#include "token_ops.h"

namespace {
enum { VX_LSE = EPI_CUSTOM, VX_DZ = EPI_CUSTOM + 1, VX_SUM = EPI_CUSTOM + 2, VX_DZ32 = EPI_CUSTOM + 3 };   // VX_DZ32: dz in fp32
constexpr int kStrip = 64;                       // columns a wave reduces in the forward pass
constexpr int kLseSplits = 16;                   // waves of the join that share a row's strips

// Reductions over a 16-lane row by rotations, one instruction a step: the rotation is an operand modifier where nothing
// hangs on the old value (bound_ctrl).  The maximum runs on integers in the floats' order (a float maximum would first
// quieten every rotated operand): negative floats have their magnitude bits flipped.
#define VX_ROR(v, n) __builtin_amdgcn_update_dpp(0, (v), 0x120 + (n), 0xf, 0xf, true)
__device__ __forceinline__ float max16(float f) {
  int v = __builtin_bit_cast(int, f);
  v ^= (v >> 31) & 0x7fffffff;
  v = max(v, VX_ROR(v, 8)); v = max(v, VX_ROR(v, 4)); v = max(v, VX_ROR(v, 2)); v = max(v, VX_ROR(v, 1));
  v ^= (v >> 31) & 0x7fffffff;
  return __builtin_bit_cast(float, v);
}
#define VX_RORF(v, n) __builtin_bit_cast(float, VX_ROR(__builtin_bit_cast(int, (v)), n))
__device__ __forceinline__ float sum16(float v) {
  v += VX_RORF(v, 8); v += VX_RORF(v, 4); v += VX_RORF(v, 2); v += VX_RORF(v, 1);
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

// What the backward pass needs of a row: p = exp(z - top) / total, so dz = exp(z - top) scaled - [label] g with scaled = g /
// total.  (exp(z - lse) would carry lse's own rounding, half a step of a value near 10, into every element of the row.)
// dz in bf16: without g, scaled = 1 / total and 1 at the label.
// Rows past the last and rows without a label have g = 0.
struct alignas(16) VxRow {
  float top, scaled, g;
  int label;                                     // -1 where the row has none, or no gradient
};

// exp(d) for d <= 0 or so with the rounding of d log2(e) made good: the product's error, up to |d| 2^-24 of the result, is
// computed and applied to first order.
__device__ __forceinline__ float exp_exact(float d) {
  const float hi = d * 1.44269502f, rest = fmaf(d, 1.92596303e-8f, fmaf(d, 1.44269502f, -hi));
  const float lo = d < -200.f ? 0.f : rest;      // there the result is 0, and of -inf the product's error is NaN
  const float e = __builtin_amdgcn_exp2f(hi);
  return fmaf(e * 0.693147181f, lo, e);
}

template <bool WHOLE, typename T>
__device__ __forceinline__ tk_u32x4 piece_of(const T* row, int c, int C) {
  if constexpr (WHOLE) return *reinterpret_cast<const tk_u32x4_at2*>(row + c);
  else return TkPiece<T, false>::load(row, c, C);
}

// Whether one of the wave's sums is infinite or NaN, and such sums taken from t
template <int I, int J>
__device__ __forceinline__ bool vx_not_finite(const f32x4 (&acc)[I][J]) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) t = fmaf(acc[i][j][r], 0.f, t);
  return __ballot(t != t) != 0;
}
template <int J>
__device__ __forceinline__ void vx_mend(f32x4 (&acc)[J], const f32x4 (&t)[J]) {
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[j][r] = fabsf(acc[j][r]) < __builtin_huge_valf() ? acc[j][r] : t[j][r];
}

struct VxGemm : DtfGemmArgs {
  // VX_LSE
  const long long* labels;
  float2* part;                                  // [strips][M]
  float2* target;                                // [M]: the label's logit, whether an earlier column of its strip reaches it
  int v0;                                        // vocabulary index of column 0
  // VX_DZ (C = dz [M, ldc], Ct = dz^T [N, ldct], null: not needed; both leading dimensions are the padded widths, padding is
  // zeroed; of fp32 operands three bf16 planes each); VX_DZ32: C in fp32
  const VxRow* rows;                             // padded to the block height; VX_SUM: each row times its g, if given
  unsigned a_plane, b_plane;                     // bytes between the planes of the operands (EPI_PLANES)
  // fp32 logits made of planes: the operands as they are ([M, D] and [N, D]); null: not made of planes
  const float* x32; const float* w32;
  long ldx32, ldw32;
  int D;
  float* db_part;                                // [wave rows][N], optional
  // VX_SUM: fp32 result C32 [splits][M, ldc32] (accumulate: added to what is there), times *scale if given; with C the
  // sum goes there as bf16 [M, ldc] instead
  const float* scale;
  int kper, accumulate;

  // The block's K range (split blockIdx.y of a grid of tiles x splits) and tile.  Workgroups go to the 8 XCDs in turn; the
  // remap over the whole grid puts the tiles of one K range next to each other on one XCD, where they share its panels.
  __device__ __forceinline__ int select() {
    const int tiles = (int)gridDim.x;
    const int lin = dtf_xcd_remap((int)(blockIdx.y * gridDim.x + blockIdx.x), tiles * (int)gridDim.y);
    const int y = lin / tiles;
    if (kper > 0) {
      const int k0 = y * kper;
      const unsigned off = (unsigned)k0 * 2u;
      A = static_cast<const char*>(A) + off;
      B = static_cast<const char*>(B) + off;
      a_bytes -= off;
      b_bytes -= off;
      K = min(kper, K - k0);
      C32 += (size_t)y * M * ldc32;
    }
    return lin - y * tiles;
  }

  // acc[ri][cj][r] = C[crow + 16 ri + 4 (lane >> 4) + r][ccol + 16 cj + (lane & 15)]; wl: 16 KB of LDS of this wave
  template <int EPI, bool F32, int RI>
  __device__ __forceinline__ void epilogue(f32x4 (&acc)[RI][4], unsigned char* wl, int crow, int ccol, int lane) const {
    if (ccol >= N) return;                       // wave-uniform: no column of this block exists
    const int fr = lane & 15, g = lane >> 4;
    if constexpr (EPI == VX_SUM) {
      store_sum<RI>(acc, wl, crow, ccol, lane);
      return;
    }
    constexpr bool kExact = F32 || EPI == VX_DZ32;
    const float NEG_INF = -__builtin_huge_valf();
    if constexpr (F32) {
#pragma unroll
      for (int ri = 0; ri < RI; ++ri)            // one home for them on both ways: else a second set of accumulators is kept
#pragma unroll
        for (int cj = 0; cj < 4; ++cj) asm volatile("" : "+v"(acc[ri][cj]));
      if (x32 && vx_not_finite(acc)) again<RI>(acc, crow, ccol, lane);
    }
    if (bias) {
#pragma unroll
      for (int cj = 0; cj < 4; ++cj) {
        const float b = ccol + 16 * cj + fr < N ? bias[ccol + 16 * cj + fr] : 0.f;
#pragma unroll
        for (int ri = 0; ri < RI; ++ri)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[ri][cj][r] += b;
      }
    }
    if (ccol + kStrip > N) {                     // only the vocabulary's last strip has columns that do not exist
#pragma unroll
      for (int cj = 0; cj < 4; ++cj)
#pragma unroll
        for (int ri = 0; ri < RI; ++ri)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[ri][cj][r] = ccol + 16 * cj + fr < N ? acc[ri][cj][r] : NEG_INF;
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
      // rows without a gradient have g = 0 and get zeros whatever p is (a padding row may hold anything)
      // The wave's rows go through its LDS (the images below overwrite them) and are read four at a time, again where a label
      // is found: held at once they would not fit beside the accumulators.
      VxRow* const lrow = reinterpret_cast<VxRow*>(wl);
#pragma unroll
      for (int k = 0; k < (16 * RI + 63) / 64; ++k)
        if (64 * k + lane < 16 * RI) lrow[64 * k + lane] = rows[crow + 64 * k + lane];
      bool any = false;                          // a row's label lies in one strip of V / 64
#pragma unroll
      for (int ri = 0; ri < RI; ++ri) {
        asm volatile("" ::: "memory");           // keeps the compiler from reading all rows up front
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const VxRow row = lrow[16 * ri + 4 * g + r];
          any |= (unsigned)(row.label - v0 - ccol) < (unsigned)kStrip;       // label -1: far below or above every strip
#pragma unroll
          for (int cj = 0; cj < 4; ++cj) {
            const float d = acc[ri][cj][r] - row.top;
            float v = (kExact ? exp_exact(d) : __expf(d)) * row.scaled;
            if (kExact) asm("" : "+v"(v));      // computed, then chosen: as a branch for every element it costs more
            acc[ri][cj][r] = row.g == 0.f ? 0.f : v;
          }
        }
      }
      if (__ballot(any)) {
#pragma unroll
        for (int ri = 0; ri < RI; ++ri) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const VxRow row = lrow[16 * ri + 4 * g + r];
            const int at = row.label - v0 - ccol - fr;
#pragma unroll
            for (int cj = 0; cj < 4; ++cj) acc[ri][cj][r] -= at == 16 * cj ? (kExact ? row.g : 1.f) : 0.f;
          }
        }
      }
      if (db_part) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ri = 0; ri < RI; ++ri) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float own = kExact ? 1.f : lrow[16 * ri + 4 * g + r].g;
#pragma unroll
            for (int cj = 0; cj < 4; ++cj) sum[cj] += kExact ? acc[ri][cj][r] : acc[ri][cj][r] * own;
          }
        }
#pragma unroll
        for (int cj = 0; cj < 4; ++cj) {
          float v = sum[cj];
          v += __shfl_xor(v, 16);
          v += __shfl_xor(v, 32);
          const int col = ccol + 16 * cj + fr;
          if (g == 0 && col < N) db_part[(size_t)(crow / (16 * RI)) * N + col] = v;
        }
      }
      if constexpr (EPI == VX_DZ32) {
        float* const c = static_cast<float*>(C);
#pragma unroll
        for (int ri = 0; ri < RI; ++ri)
#pragma unroll
          for (int cj = 0; cj < 4; ++cj)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int row = crow + 16 * ri + 4 * g + r, col = ccol + 16 * cj + fr;
              if (row < M && col < ldc) c[(size_t)row * ldc + col] = acc[ri][cj][r];
            }
      } else {
        if constexpr (!F32) {
          store_dz<RI, false>(acc, wl, crow, ccol, lane, 0);
        } else {
#pragma unroll 1                                 // three planes at once would not fit the registers
          for (int q = 0; q < 3; ++q) {
            int l = lane;
            asm volatile("" : "+v"(l));          // addresses are computed plane by plane, not kept
            store_dz<RI, true>(acc, wl, crow, ccol, l, q);
          }
        }
      }
    }
  }

  // The block's sums again, with fp32 instructions: a lane's 16-byte piece of a row is the operand of four.  Rows and columns
  // past the last repeat it.  Two tiles of 16 rows at a time: all of them would cost the kernel a wave's registers.
  template <int RI>
  __device__ __forceinline__ void again(f32x4 (&acc)[RI][4], int crow, int ccol, int lane) const {
    constexpr int H = RI > 1 ? 2 : 1;
    const int fr = lane & 15, g = lane >> 4;
    const float* b_row[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b_row[j] = w32 + (long)min(ccol + 16 * j + fr, N - 1) * ldw32;
    unrolled<0, RI / H>([&](auto Half) {
      constexpr int i0 = Half * H;
      f32x4 t[H][4];
#pragma unroll
      for (int i = 0; i < H; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) t[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int k0 = 0; k0 < D; k0 += 16) {
        tk_u32x4 b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = piece_of<false>(b_row[j], k0 + 4 * g, D);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const tk_u32x4 a = piece_of<false>(x32 + (long)min(crow + 16 * (i0 + i) + fr, M - 1) * ldx32, k0 + 4 * g, D);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              t[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[j][e]), t[i][j], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < H; ++i) vx_mend(acc[i0 + i], t[i]);
    });
  }

  // Both images are turned in LDS, so that every global store is 16 bytes a lane.
  template <int RI, bool PLANES>
  __device__ __forceinline__ void store_dz(f32x4 (&acc)[RI][4], unsigned char* wl, int crow, int ccol, int lane, int plane) const {
    constexpr int CH = 2 * RI;                   // 16-byte chunks of a transposed row (16 RI rows of dz)
    const int fr = lane & 15, g = lane >> 4;
    unsigned short* const c = static_cast<unsigned short*>(C) + (size_t)plane * M * ldc;
    unsigned short* const ct = static_cast<unsigned short*>(Ct) + (size_t)plane * N * ldct;
    uint2 pk[RI][4];
#pragma unroll
    for (int ri = 0; ri < RI; ++ri)
#pragma unroll
      for (int cj = 0; cj < 4; ++cj) {
        pk[ri][cj].x = tk_pack2(acc[ri][cj][0], acc[ri][cj][1]);
        pk[ri][cj].y = tk_pack2(acc[ri][cj][2], acc[ri][cj][3]);
        if (PLANES) {                            // what the next planes hold; now, so that nothing else stays alive
          acc[ri][cj][0] -= __uint_as_float(pk[ri][cj].x << 16); acc[ri][cj][1] -= __uint_as_float(pk[ri][cj].x & 0xffff0000u);
          acc[ri][cj][2] -= __uint_as_float(pk[ri][cj].y << 16); acc[ri][cj][3] -= __uint_as_float(pk[ri][cj].y & 0xffff0000u);
          asm volatile("" : "+v"(acc[ri][cj]));
        }
      }
    if (Ct) {
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
    }
    if (!C) return;
    // straight image: neighbouring lanes swap halves, so that a lane holds two rows of two neighbouring columns and writes
    // 32-bit pieces (even lanes rows 0 and 1 of the four, odd lanes rows 2 and 3)
    const bool odd = fr & 1;
    const unsigned lo_sel = odd ? 0x05040100u : 0x01000504u, hi_sel = odd ? 0x07060302u : 0x03020706u;
    // row 16 ri + 4 g + {0, 2}, 16-byte chunk (2 cj + fr / 8) ^ (row / 4): ri adds 2048 bytes and flips bit 2 of the chunk
    const unsigned at0 = (unsigned)(4 * g + (odd ? 2 : 0)) * 128u + (unsigned)(fr & 6) * 2u, ch0 = (unsigned)((fr >> 3) ^ g);
#pragma unroll
    for (int cj = 0; cj < 4; ++cj) {
      unsigned char* const even_ri = wl + at0 + ((ch0 ^ (2 * cj)) << 4);
      unsigned char* const odd_ri = wl + at0 + ((ch0 ^ (2 * cj) ^ 4) << 4);
#pragma unroll
      for (int ri = 0; ri < RI; ++ri) {
        const unsigned send = odd ? pk[ri][cj].x : pk[ri][cj].y, own = odd ? pk[ri][cj].y : pk[ri][cj].x;
        const unsigned got = (unsigned)__builtin_amdgcn_update_dpp(0, (int)send, 0xB1, 0xf, 0xf, true);     // lane ^ 1
        unsigned* const at = reinterpret_cast<unsigned*>((ri & 1 ? odd_ri : even_ri) + 2048 * ri);
        at[0] = __builtin_amdgcn_perm(own, got, lo_sel);
        at[32] = __builtin_amdgcn_perm(own, got, hi_sel);
      }
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
            const float own = rows ? f * rows[row].g : f;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= own;
          }
          if (c16) *reinterpret_cast<uint2*>(&c16[(size_t)row * ldc + col]) = make_uint2(tk_pack2(v[0], v[1]), tk_pack2(v[2], v[3]));
          else *p = v;
        }
      }
    }
  }
};

// The kernels of few rows.  Loads in their loops carry no conditions, which would keep the compiler from having several under
// way: rows and steps past the last repeat it (their results are not stored, their products left out, or they meet zeros),
// and waves whose pieces are all WHOLE have a loop of their own that does not look at the row's end.
// The four waves' sums of a workgroup, in wave 0
template <int RT>
__device__ __forceinline__ void vx_join_waves(float (&s)[3][16 * RT][64], f32x4 (&acc)[RT][4], int wave, int lane) {
  if (wave) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[wave - 1][16 * i + 4 * j + r][lane] = acc[i][j][r];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 16 * i + 4 * j + r;
        acc[i][j][r] = ((acc[i][j][r] + s[0][at][lane]) + s[1][at][lane]) + s[2][at][lane];
      }
}

// Few rows, or few columns: 16 rows x 64 columns a workgroup, the four waves share K (64 bytes of a row a step, wave by wave),
// operands straight from memory into the matrix instructions: one wave's 20 loads in flight, no staging, no barrier in the
// loop.  Every row of W is read by ceil(M / 16) workgroups, next to each other on one XCD.
// Not ALIGNED (fp32 only): rows of any width, stride and alignment, the elements behind a row's end replaced by zeros.
template <typename T, int EPI, bool ALIGNED>
__global__ __launch_bounds__(256, 4) void vx_skinny_kernel(VxGemm p) {
  typedef std::conditional_t<sizeof(T) == 4, float, unsigned short> E;
  constexpr int PER16 = Elem<T>::PER16, AHEAD = 4;
  __shared__ __attribute__((aligned(16))) float s_acc[3][16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, g = lane >> 4;
  const int tiles_m = (p.M + 15) >> 4, wg = dtf_xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = (wg % tiles_m) * 16, n0 = (wg / tiles_m) * 64;
  const rsrc_t ra = make_rsrc(p.A, p.a_bytes), rb = make_rsrc(p.B, p.b_bytes);
  // rows and columns past the last repeat it: the epilogue leaves them out
  const int row = min(m0 + fr, p.M - 1);
  const unsigned a_off = (unsigned)row * (unsigned)p.lda * (unsigned)sizeof(T);
  const E* const a_row = static_cast<const E*>(p.A) + (long)row * p.lda;
  unsigned b_off[4];
  const E* b_row[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = min(n0 + 16 * j + fr, p.N - 1);
    b_off[j] = (unsigned)col * (unsigned)p.ldb * (unsigned)sizeof(T);
    b_row[j] = static_cast<const E*>(p.B) + (long)col * p.ldb;
  }
  f32x4 acc[1][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // steps of 4 pieces of 16 bytes: all of them if ALIGNED (pieces past the end are out of the buffer's range and read as zeros),
  // else the whole ones, and the rest below
  const int steps = ALIGNED ? (p.K + 4 * PER16 - 1) / (4 * PER16) : p.K / (4 * PER16);
  for (int s = wave; s < steps; s += 4 * AHEAD) {
    u32x4 a[AHEAD], b[AHEAD][4];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = min(s + 4 * u, steps - 1) * 4 + g;       // 16-byte piece of the row
      if constexpr (ALIGNED) {
        const bool in = k * PER16 < p.K;
        a[u] = __builtin_amdgcn_raw_buffer_load_b128(ra, (int)(in ? a_off + k * 16u : kOOB), 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) b[u][j] = __builtin_amdgcn_raw_buffer_load_b128(rb, (int)(in ? b_off[j] + k * 16u : kOOB), 0, 0);
      } else {
        a[u] = piece_of<true>(a_row, k * PER16, p.K);
#pragma unroll
        for (int j = 0; j < 4; ++j) b[u][j] = piece_of<true>(b_row[j], k * PER16, p.K);
      }
    }
    __builtin_amdgcn_sched_barrier(0);           // all loads under way before the first product
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (s + 4 * u >= steps) break;               // the same for the whole wave
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_slot<T>(a[u], b[u][j], acc[0][j]);
    }
  }
  if (!ALIGNED && wave == (steps & 3) && steps * 4 * PER16 < p.K) {
    const int k = (steps * 4 + g) * PER16;
    const u32x4 a = k < p.K ? piece_of<false>(a_row, k, p.K) : tk_u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 4; ++j) mma_slot<T>(a, k < p.K ? piece_of<false>(b_row[j], k, p.K) : tk_u32x4{0u, 0u, 0u, 0u}, acc[0][j]);
  }
  vx_join_waves<1>(s_acc, acc, wave, lane);
  if (wave) return;
  // the epilogue's 2 KB: memory that this wave, the only one left, has just read
  p.template epilogue<EPI, sizeof(T) == 4>(acc, reinterpret_cast<unsigned char*>(s_acc), m0, n0, lane);
}

// The products of few rows (few_rows), straight from X, W and the fp32 dz, with fp32 matrix instructions: the time goes
// into reading W and writing dW once, so no transposed copies and no planes are made.  A lane's 16-byte piece of a row of W
// (or X) is the operand of VEC instructions at once: instruction q takes column c0 + VEC fr + q.

// dX: workgroup (column tile, 16 RT rows, range of the vocabulary); the waves take 16 vocabulary rows each in turn.
// ROUND: fp32 weights under bf16 activations, rounded as the logits' copy of them was.
template <typename T, bool ROUND, int RT>
__global__ __launch_bounds__(256) void vx_small_dx_kernel(const float* __restrict__ dz, long lddz, const T* __restrict__ w, long ldw, float* __restrict__ out,
                                                          int M, int D, long n, int per, int ldo) {
  typedef TkPiece<T, false> P;
  constexpr int VEC = P::VEC;
  __shared__ float s_acc[3][4 * VEC * RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, g = lane >> 4;
  const int c = (int)blockIdx.x * 16 * VEC + VEC * fr, cc = c < D ? c : 0, m0 = blockIdx.y * 16 * RT;
  // n is below 2^30; a wave's first 16 vocabulary rows of the range, and the last 16 it may reach
  const int lo = (int)min((long)blockIdx.z * per, n), hi = (int)min(n, (long)lo + per), first = lo + 16 * wave, last = (hi - 1) & ~15;
  f32x4 acc[RT][VEC];
  const float* arow[RT];                         // rows past the last repeat it and are not stored
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    arow[i] = dz + (long)min(m0 + 16 * i + fr, M - 1) * lddz;
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  constexpr int AHEAD = 2;
  struct Pieces { f32x4 a[AHEAD][RT]; tk_u32x4 b[AHEAD][4]; };
  auto run = [&](auto whole) {
    auto load = [&](int v, Pieces& t) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int at = min(v + 64 * u, last) + 4 * g;        // dz is zero from n to its padded width, a multiple of 64 columns
#pragma unroll
        for (int i = 0; i < RT; ++i) t.a[u][i] = *reinterpret_cast<const f32x4*>(arow[i] + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) t.b[u][j] = piece_of<decltype(whole)::value>(w + (long)min(at + j, hi - 1) * ldw, cc, D);
      }
      __builtin_amdgcn_sched_barrier(0);         // all loads under way before the first product
    };
    auto product = [&](int v, const Pieces& t) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (v + 64 * u >= hi) break;             // the same for the whole wave
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float wv[VEC];
          P::unpack(t.b[u][j], wv);
#pragma unroll
          for (int q = 0; q < VEC; ++q) {
            if (ROUND) wv[q] = tk_bf2f(tk_f2bf(wv[q]));
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[i][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(t.a[u][i][j], wv[q], acc[i][q], 0, 0, 0);
          }
        }
      }
    };
    for (int v = first; v < hi; v += 64 * AHEAD) {
      Pieces t;
      load(v, t);
      product(v, t);
    }
  };
  if (first < hi) {
    if (__ballot(cc + VEC > D) == 0) run(std::true_type{});
    else run(std::false_type{});
  }
  if (wave) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int q = 0; q < VEC; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_acc[wave - 1][4 * (VEC * i + q) + r][lane] = acc[i][q][r];
  }
  __syncthreads();
  if (wave || c >= ldo) return;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = m0 + 16 * i + 4 * g + r;
      if (row >= M) continue;
      float* const o = out + ((size_t)blockIdx.z * M + row) * ldo + c;
#pragma unroll
      for (int q = 0; q < VEC; q += 4) {
        f32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = 4 * (VEC * i + q + e) + r;
          t[e] = ((acc[i][q + e][r] + s_acc[0][at][lane]) + s_acc[1][at][lane]) + s_acc[2][at][lane];
        }
        if (c + q < ldo) *reinterpret_cast<f32x4*>(o + q) = t;
      }
    }
}

// dW: a wave owns 16 RT vocabulary rows and 16 VEC columns; the waves of a workgroup have the columns in common.
template <typename TX, typename TO, int RT>
__global__ __launch_bounds__(256, RT > 1 ? 3 : 1) void vx_small_dw_kernel(const float* __restrict__ dz, long lddz, const TX* __restrict__ x, long ldx, TO* __restrict__ out,
                                                          int M, int D, long n, const VxRow* __restrict__ rows, const float* __restrict__ scale) {
  typedef TkPiece<TX, false> P;
  constexpr int VEC = P::VEC, OUT = 16 / sizeof(TO);
  const int lane = threadIdx.x & 63, fr = lane & 15, g = lane >> 4;
  const int tiles = (D + 16 * VEC - 1) / (16 * VEC);
  const long v0 = (long)(blockIdx.x / tiles) * 64 * RT + 16 * RT * (threadIdx.x >> 6);
  const int c = (int)(blockIdx.x % tiles) * 16 * VEC + VEC * fr;
  f32x4 acc[RT][VEC];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int cc = c < D ? c : 0;
  const float* col[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) col[i] = dz + min(v0 + 16 * i + fr, n - 1);
  auto run = [&](auto whole) {
    for (int k = 0; k < M; k += 16) {
      float a[4][RT], gr[4];
      tk_u32x4 b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = min(k + 4 * u + g, M - 1);
        gr[u] = rows[row].g;
#pragma unroll
        for (int i = 0; i < RT; ++i) a[u][i] = col[i][(long)row * lddz];
        b[u] = piece_of<decltype(whole)::value>(x + (long)row * ldx, cc, D);
        if (k + 4 * u + g >= M) gr[u] = 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);         // all loads under way before the first product
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float xv[VEC];
        P::unpack(b[u], xv);
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const float xq = gr[u] != 0.f ? xv[q] : 0.f;         // (see vx_transpose_kernel)
#pragma unroll
          for (int i = 0; i < RT; ++i) acc[i][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][i], xq, acc[i][q], 0, 0, 0);
        }
      }
    }
  };
  if (__ballot(cc + VEC > D) == 0) run(std::true_type{});
  else run(std::false_type{});
  const float f = *scale;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long v = v0 + 16 * i + 4 * g + r;
      if (v >= n) continue;
#pragma unroll
      for (int q = 0; q < VEC; q += OUT) {
        float t[OUT];
#pragma unroll
        for (int e = 0; e < OUT; ++e) t[e] = acc[i][q + e][r] * f;
        if (c + q < D) TkPiece<TO, false>::store(out + v * D, c + q, D, t);
      }
    }
}

// The fp32 kernels of 17 rows and more: operands as they are in memory, cut into their three bf16 planes in registers, six
// products of planes with the bf16 matrix instructions (96 cycles for 16 x 16 x 32 where fp32's take 256).  The next step's
// loads are on their way during the products.
struct VxSplit { bf16x8_t p[3]; };
__device__ __forceinline__ VxSplit vx_split(const float (&v)[8]) {
  VxSplit s;
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = tk_pack2(r[2 * e], r[2 * e + 1]);
      r[2 * e] -= __uint_as_float(w[e] << 16);
      r[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
    }
    s.p[q] = __builtin_bit_cast(bf16x8_t, w);
  }
  return s;
}
template <int RT>
__device__ __forceinline__ void vx_split_product(const VxSplit (&a)[RT], const VxSplit (&b)[4], f32x4 (&acc)[RT][4]) {
  constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};        // the small products first
#pragma unroll
  for (int k = 0; k < 6; ++k)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i].p[PA[k]], b[j].p[PB[k]], acc[i][j], 0, 0, 0);
}
__device__ __forceinline__ void vx_eight(const tk_u32x4 (&q)[2], float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(q[e >> 2][e & 3]);
}
// Logits: 16 RT rows x 64 columns a workgroup, the waves take 32 elements of K each in turn (a lane 32 bytes of a row).
template <int EPI, int RT>
__global__ __launch_bounds__(256, 2) void vx_split_logits_kernel(VxGemm p) {
  __shared__ __attribute__((aligned(16))) float s_acc[3][16 * RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, g = lane >> 4;
  const int tiles_m = (p.M + 16 * RT - 1) / (16 * RT), wg = dtf_xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = (wg % tiles_m) * 16 * RT, n0 = (wg / tiles_m) * 64;
  const float* a_row[RT];                        // rows and columns past the last repeat it: the epilogue leaves them out
  const float* b_row[4];
#pragma unroll
  for (int i = 0; i < RT; ++i) a_row[i] = static_cast<const float*>(p.A) + (long)min(m0 + 16 * i + fr, p.M - 1) * p.lda + 8 * g;
#pragma unroll
  for (int j = 0; j < 4; ++j) b_row[j] = static_cast<const float*>(p.B) + (long)min(n0 + 16 * j + fr, p.N - 1) * p.ldb + 8 * g;
  f32x4 acc[RT][4];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = p.K >> 5;                    // whole ones; the rest below
  tk_u32x4 a[RT][2], b[4][2];
  auto load = [&](int s) {
    const int k = min(s, steps - 1) * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j][h] = piece_of<true>(b_row[j], k + 4 * h, p.K);
#pragma unroll
      for (int i = 0; i < RT; ++i) a[i][h] = piece_of<true>(a_row[i], k + 4 * h, p.K);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  VxSplit sa[RT], sb[4];
  auto split = [&] {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) { vx_eight(b[j], v); sb[j] = vx_split(v); }
#pragma unroll
    for (int i = 0; i < RT; ++i) { vx_eight(a[i], v); sa[i] = vx_split(v); }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (wave < steps) {
    load(wave);
    for (int s = wave; s < steps; s += 4) {
      split();
      load(s + 4);
      vx_split_product<RT>(sa, sb, acc);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (wave == (steps & 3) && steps * 32 < p.K) {
    const int k = steps * 32, left = p.K - k - 8 * g;        // elements of this lane's eight that exist
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j][h] = 4 * h < left ? piece_of<false>(b_row[j] + k, 4 * h, left) : tk_u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < RT; ++i) a[i][h] = 4 * h < left ? piece_of<false>(a_row[i] + k, 4 * h, left) : tk_u32x4{0u, 0u, 0u, 0u};
    }
    split();
    vx_split_product<RT>(sa, sb, acc);
  }
  vx_join_waves<RT>(s_acc, acc, wave, lane);
  if (wave) return;
  // the epilogue's 2 KB a tile: memory that this wave, the only one left, has just read
  p.template epilogue<EPI, true>(acc, reinterpret_cast<unsigned char*>(s_acc), m0, n0, lane);
}

// dX: workgroup (64 columns, 16 RT rows, range of the vocabulary); the waves take 32 vocabulary rows each in turn, a lane eight of
// them and four columns.
template <int RT>
__global__ __launch_bounds__(256, 2) void vx_split_dx_kernel(const float* __restrict__ dz, long lddz, const float* __restrict__ w, long ldw, float* __restrict__ out,
                                                             int M, int D, long n, int per, int ldo) {
  __shared__ float s_acc[3][16 * RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, g = lane >> 4;
  const int c = (int)blockIdx.x * 64 + 4 * fr, cc = c < D ? c : 0, m0 = blockIdx.y * 16 * RT;
  // n is below 2^30; a wave's first 32 vocabulary rows of the range, and the last 32 it may reach
  const int lo = (int)min((long)blockIdx.z * per, n), hi = (int)min(n, (long)lo + per), first = lo + 32 * wave, last = (hi - 1) & ~31;
  f32x4 acc[RT][4];
  const float* arow[RT];                         // rows past the last repeat it and are not stored
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    arow[i] = dz + (long)min(m0 + 16 * i + fr, M - 1) * lddz;
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto run = [&](auto whole) {
    tk_u32x4 a[RT][2], b[8];
    auto load = [&](int v) {
      const int at = min(v, last) + 8 * g;       // dz is zero from n to its padded width, a multiple of 64 columns
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = piece_of<decltype(whole)::value>(w + (long)min(at + j, hi - 1) * ldw, cc, D);
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) a[i][h] = *reinterpret_cast<const tk_u32x4*>(arow[i] + at + 4 * h);
      __builtin_amdgcn_sched_barrier(0);
    };
    load(first);
    for (int v = first; v < hi; v += 128) {
      VxSplit sa[RT], sb[4];
      float e[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = __uint_as_float(b[j][q]);
        sb[q] = vx_split(e);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) { vx_eight(a[i], e); sa[i] = vx_split(e); }
      __builtin_amdgcn_sched_barrier(0);
      load(v + 128);
      vx_split_product<RT>(sa, sb, acc);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (first < hi) {
    if (__ballot(cc + 4 > D) == 0) run(std::true_type{});
    else run(std::false_type{});
  }
  if (vx_not_finite(acc))                        // (see the head of this file)
    unrolled<0, RT>([&](auto I) {
      f32x4 t[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int v = first; v < hi; v += 128)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = v + 8 * g + j;
          const float e = arow[I][at];
          const tk_u32x4 b = piece_of<false>(w + (long)min(at, hi - 1) * ldw, cc, D);
#pragma unroll
          for (int q = 0; q < 4; ++q) t[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(e, __uint_as_float(b[q]), t[q], 0, 0, 0);
        }
      vx_mend(acc[I], t);
    });
  vx_join_waves<RT>(s_acc, acc, wave, lane);
  if (wave || c >= ldo) return;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = m0 + 16 * i + 4 * g + r;
      if (row < M) *reinterpret_cast<f32x4*>(out + ((size_t)blockIdx.z * M + row) * ldo + c) = f32x4{acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
    }
}

// dW: a wave owns 64 vocabulary rows and 64 columns, 32 rows of X a step.
__global__ __launch_bounds__(256, 2) void vx_split_dw_kernel(const float* __restrict__ dz, long lddz, const float* __restrict__ x, long ldx, float* __restrict__ out,
                                                             int M, int D, long n, const VxRow* __restrict__ rows, const float* __restrict__ scale) {
  const int lane = threadIdx.x & 63, fr = lane & 15, g = lane >> 4;
  const int tiles = (D + 63) / 64;
  const long v0 = (long)(blockIdx.x / tiles) * 256 + 64 * (threadIdx.x >> 6);
  const int c = (int)(blockIdx.x % tiles) * 64 + 4 * fr, cc = c < D ? c : 0;
  f32x4 acc[4][4];
  const float* col[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    col[i] = dz + min(v0 + 16 * i + fr, n - 1);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto run = [&](auto whole) {
    for (int k = 0; k < M; k += 32) {
      float a[4][8], gr[8];
      tk_u32x4 b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = min(k + 8 * g + j, M - 1);
        gr[j] = rows[row].g;
        b[j] = piece_of<decltype(whole)::value>(x + (long)row * ldx, cc, D);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i][j] = col[i][(long)row * lddz];
        if (k + 8 * g + j >= M) gr[j] = 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);         // all loads under way before the first product
      VxSplit sa[4], sb[4];
      float e[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = gr[j] != 0.f ? __uint_as_float(b[j][q]) : 0.f;      // (see vx_transpose_kernel)
        sb[q] = vx_split(e);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i] = vx_split(a[i]);
      vx_split_product<4>(sa, sb, acc);
    }
  };
  if (__ballot(cc + 4 > D) == 0) run(std::true_type{});
  else run(std::false_type{});
  if (vx_not_finite(acc))                        // (see the head of this file)
    unrolled<0, 4>([&](auto I) {
      f32x4 t[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int k = 0; k < M; k += 4) {
        const int row = min(k + g, M - 1);
        const bool in = k + g < M && rows[row].g != 0.f;
        const float e = k + g < M ? col[I][(long)row * lddz] : 0.f;
        const tk_u32x4 b = piece_of<false>(x + (long)row * ldx, cc, D);
#pragma unroll
        for (int q = 0; q < 4; ++q) t[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(e, in ? __uint_as_float(b[q]) : 0.f, t[q], 0, 0, 0);
      }
      vx_mend(acc[I], t);
    });
  const float f = *scale;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long v = v0 + 16 * i + 4 * g + r;
      if (v >= n || c >= D) continue;
      const float t[4] = {acc[i][0][r] * f, acc[i][1][r] * f, acc[i][2][r] * f, acc[i][3][r] * f};
      TkPiece<float, false>::store(out + v * D, c, D, t);
    }
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

// dst[c, r] = src[r, c] for r < M, c < N; zeros for r in [M, ldt) and, of X (rows given), for rows without a gradient: in dW
// they meet dz = 0, and a padding row that holds NaN or infinities must not make a sum of it.  64 x 64 tiles through LDS.
// weighted: X times the row's g, rounded to bf16 (each element by its own half step at most, no direction in common).
__global__ __launch_bounds__(256) void vx_transpose_kernel(const unsigned short* __restrict__ src, unsigned short* __restrict__ dst, int M, int N, long lds_, int ldt,
                                                           const VxRow* __restrict__ rows, int weighted) {
  __shared__ unsigned short tile[64][72];
  const int across = (N + 63) >> 6, c0 = (int)(blockIdx.x % across) * 64, r0 = (int)(blockIdx.x / across) * 64;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int id = threadIdx.x + 256 * i, rr = id >> 3, ch = id & 7;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (r0 + rr < M && c0 + ch * 8 < N && !(rows && rows[r0 + rr].g == 0.f)) v = *reinterpret_cast<const u32x4*>(src + (size_t)(r0 + rr) * lds_ + c0 + ch * 8);
    if (weighted && r0 + rr < M) {
      const float own = rows[r0 + rr].g;
      float f[8];
      TkVec<unsigned short, 8>::unpack(v, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= own;
      v = TkVec<unsigned short, 8>::pack(f);
    }
    *reinterpret_cast<u32x4*>(&tile[rr][ch * 8]) = v;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int id = threadIdx.x + 256 * i, cc = id >> 3, ch = id & 7;
    if (c0 + cc >= N || r0 + ch * 8 >= ldt) continue;
    unsigned e[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = (unsigned)tile[ch * 8 + 2 * k][cc] | ((unsigned)tile[ch * 8 + 2 * k + 1][cc] << 16);
    *reinterpret_cast<u32x4*>(dst + (size_t)(c0 + cc) * ldt + r0 + ch * 8) = u32x4{e[0], e[1], e[2], e[3]};
  }
}

// Nearest bf16, but the largest finite one for finite numbers beyond it: 0 times such an element stays 0.
__device__ __forceinline__ unsigned short vx_first_plane(float v) {
  const unsigned short q = tk_f2bf(v);
  return (q & 0x7fff) == 0x7f80 && fabsf(v) < __builtin_huge_valf() ? q - 1 : q;
}

// The three bf16 planes of an fp32 matrix [M, N] (any stride and alignment), straight [3][M, Np] and / or transposed
// [3][Nt, Mp], zeros in the padding; in the transposed one also for rows without a gradient (see vx_transpose_kernel).
// Two matrices a launch: those of a small X are latency only, beside W's they cost nothing.
struct VxPlanes {
  const float* src; unsigned short* dst; unsigned short* dst_t; const VxRow* rows;
  long lds_; int M, N, Np, Nt, Mp, blocks;
};
__global__ __launch_bounds__(256) void vx_planes_kernel(VxPlanes first, VxPlanes second) {
  const bool one = (int)blockIdx.x < first.blocks;
  const float* const src = one ? first.src : second.src;
  unsigned short* const dst = one ? first.dst : second.dst;
  unsigned short* const dst_t = one ? first.dst_t : second.dst_t;
  const VxRow* const rows = one ? first.rows : second.rows;
  const long lds_ = one ? first.lds_ : second.lds_;
  const int M = one ? first.M : second.M, N = one ? first.N : second.N, Np = one ? first.Np : second.Np, Nt = one ? first.Nt : second.Nt, Mp = one ? first.Mp : second.Mp;
  const int block = (int)blockIdx.x - (one ? 0 : first.blocks);
  __shared__ float tile[64][65];
  const int across = (Np + 63) >> 6, c0 = block % across * 64, r0 = block / across * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int rr = ty + 4 * i;
    tile[rr][tx] = r0 + rr < M && c0 + tx < N ? src[(size_t)(r0 + rr) * lds_ + c0 + tx] : 0.f;
  }
  __syncthreads();
  const int ch = threadIdx.x & 7, line = threadIdx.x >> 3;          // 8 elements of a row of the result
#pragma unroll
  for (int turn = 0; turn < 2; ++turn) {
    unsigned short* const out = turn ? dst_t : dst;
    if (!out) continue;
    const long ld = turn ? Mp : Np, lines = turn ? Nt : M, plane = lines * ld;
    const int at = (turn ? r0 : c0) + ch * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int l = line + 32 * i, row = (turn ? c0 : r0) + l;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = turn ? tile[ch * 8 + k][l] : tile[l][ch * 8 + k];
        if (turn && rows && at + k < M && rows[at + k].g == 0.f) v[k] = 0.f;
      }
      if (row < lines && at < ld) {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          unsigned e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned short lo = vx_first_plane(v[2 * k]), hi = vx_first_plane(v[2 * k + 1]);
            e[k] = (unsigned)lo | ((unsigned)hi << 16);
            const float dl = v[2 * k] - tk_bf2f(lo), dh = v[2 * k + 1] - tk_bf2f(hi);
            v[2 * k] = fabsf(dl) < __builtin_huge_valf() ? dl : 0.f;
            v[2 * k + 1] = fabsf(dh) < __builtin_huge_valf() ? dh : 0.f;
          }
          *reinterpret_cast<u32x4*>(out + q * plane + row * ld + at) = u32x4{e[0], e[1], e[2], e[3]};
        }
      }
    }
  }
}

// out[r, c] = scale [* the row's g] * sum of the splits' fp32 results, in their order, rounded to the output's type.
template <typename T>
__global__ __launch_bounds__(256) void vx_finish_kernel(const float* __restrict__ ws, int splits, int rows, int cols, int ldw, T* __restrict__ out, long ldo,
                                                        const float* __restrict__ scale, const VxRow* __restrict__ own) {
  const int quads = (cols + 3) >> 2;
  const long i = (long)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  const int c = (int)(i - row * quads) * 4;
  if (row >= rows) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; s += 8) {          // eight loads under way at once (past the end: the last again, not added)
    f32x4 o[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) o[u] = *reinterpret_cast<const f32x4*>(ws + ((size_t)min(s + u, splits - 1) * rows + row) * ldw + c);
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += s + u < splits ? o[u][e] : 0.f;
  }
  const float f = own ? *scale * own[row].g : *scale;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < cols) tk_put(out + row * ldo + c + e, v[e] * f);
}

// db[c] = scale * sum of the wave rows' partial column sums
__global__ __launch_bounds__(256) void vx_db_kernel(const float* __restrict__ part, int nparts, int N, float* __restrict__ db, const float* __restrict__ scale) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float v = 0.f;
  for (int p = 0; p < nparts; ++p) v += part[(size_t)p * N + c];
  db[c] = v * *scale;
}

__device__ __forceinline__ bool vx_has_label(long long lab, long long ignore, long V) { return lab != ignore && lab >= 0 && lab < V; }

// *scale = the largest finite |dloss| of a row with a label, 1 if there is none but zeros.
__global__ __launch_bounds__(1024) void vx_largest_kernel(const float* __restrict__ dloss, const long long* __restrict__ labels, int M, long V, long long ignore,
                                                          float* __restrict__ scale) {
  __shared__ float s[16];
  float m = 0.f;
  for (int r = threadIdx.x; r < M; r += 1024) {
    const float v = fabsf(dloss[r]);
    if (vx_has_label(labels[r], ignore, V) && v < __builtin_huge_valf()) m = fmaxf(m, v);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) m = fmaxf(m, s[w]);
  *scale = m > 0.f ? m : 1.f;
}

// apart (dz in bf16): g stays out of dz; of gradients a row it is relative to *scale, which vx_largest_kernel has left.
__global__ __launch_bounds__(256) void vx_rows_kernel(const float* __restrict__ top, const float* __restrict__ total, const long long* __restrict__ labels, const float* __restrict__ dloss,
                                                      int dloss_rows, const long long* __restrict__ counts, int mean, int M, int Mp, long V,
                                                      long long ignore, int apart, VxRow* __restrict__ rows, float* __restrict__ scale) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r == 0 && !(apart && dloss_rows)) {
    const float up = dloss && !dloss_rows ? *dloss : 1.f;
    *scale = mean ? (counts[1] ? up / (float)counts[1] : 0.f) : up;
  }
  if (r >= Mp) return;
  VxRow o = {0.f, 0.f, 0.f, -1};
  if (r < M) {
    const long long lab = labels[r];
    if (vx_has_label(lab, ignore, V)) {
      o.top = top[r];
      o.g = !dloss_rows ? 1.f : apart ? dloss[r] / *scale : dloss[r];
      o.scaled = (apart ? 1.f : o.g) / total[r];
      if (o.g != 0.f) o.label = (int)lab;
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
  float* lse; float* top; float* total; float* loss_rows; float* loss; long long* counts; float* blk_loss; int* blk_counts;
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
    a.top[row] = m;
    a.total[row] = s;
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

// 256x256 blocks of the 8-wave kernel (its staging offsets ask for whole half-tiles in range): one block a CU at 1300 TFLOP/s
// of the whole chip against 450-600 of the 128x128 blocks, so from about 7/16 of the CUs on if the K loop is deep, from 3/4
// on else.
bool use_pp(int planes, long m, long n, long k, int splits) {
  const long blocks = ((m + 255) / 256) * ((n + 255) / 256) * splits, deep = k / splits * (planes == 3 ? 6 : 1);
  return m >= 256 && n >= 256 && k / splits >= 256 && blocks >= (deep >= 2048 ? 112 : 192);
}

// Up to so many rows the products read W and X as they are.  Forward and backward, this way / through transposed copies and
// planes: bf16 at 65536 x 4096, 48 rows 0.86 / 0.87 ms, 64 rows 0.98 / 0.88; fp32 at 30000 x 1024, 256 rows 0.57 / 0.70 ms, 400
// 0.83 / 0.84, 512 0.97 / 0.85; at 10000 x 512, 300 rows 185 / 209 us, 512 rows 245 / 258.
bool few_rows(int dtype, long m) { return m <= (dtype == TK_BF16 ? 32 : 448); }

// Logits by the kernel that shares K between the waves: where 128x128 blocks would leave most CUs idle or, with few rows, be
// mostly empty (bf16: as long as W is small; a large one streams faster through the 128x128 blocks: 131072 x 4096, one row,
// 203 against 227 us); fp32 with few rows always, and where the planes' 256x256 blocks would be too few (a
// shallow K leaves most of the kernel's time to the epilogue, which one wave of four does here): 1176 x 3000 x 300 forward and
// backward 163 us, through planes 181.
bool use_skinny(int dtype, long m, long n, long k) {
  const long blocks = ((m + 127) / 128) * ((n + 127) / 128);
  if (dtype == TK_BF16) return blocks < 128 || (m <= 16 && blocks < 512);
  return blocks < 128 || few_rows(dtype, m) || (k >= 256 && !use_pp(3, m, n, k, 1));
}

// fp32 logits from planes: where the kernel above does not take them.
bool use_planes(int dtype, bool skinny) { return dtype == TK_F32 && !skinny; }

// Tiles of 16 rows that one workgroup of the fp32 kernels of few rows takes (each element of W it reads and cuts serves all of
// them), while two workgroups a CU are left.  Forward and backward: 64 rows at 65536 x 4096, one tile (fp32 instructions) 2.17 ms,
// two 1.45, four 1.25; 140 rows at 30000 x 1024, two 0.53, four 0.41.  (bf16: two tiles at 32 rows made no difference.)
int row_tiles(int dtype, long m, long others) {
  for (int rt = dtype == TK_BF16 ? 1 : 4; rt > 1; rt /= 2)
    if (m > 8 * rt && (m + 16 * rt - 1) / (16 * rt) * others >= 512) return rt;
  return 1;
}
int skinny_tiles(int dtype, long m, long n) { return row_tiles(dtype, m, (n + 63) / 64); }

// Rows of a wave's block in the logits' epilogue
int wave_rows(const VxGemm& a, bool skinny) {
  return skinny ? 16 * skinny_tiles(a.dtype, a.M, a.N) : use_pp(a.a_plane ? 3 : 1, a.M, a.N, a.K, 1) ? 128 : 64;
}

template <int EPI>
void launch_gemm(const VxGemm& a, int splits, hipStream_t s) {
  const bool planes = a.a_plane > 0;
  if (use_pp(planes ? 3 : 1, a.M, a.N, a.K, splits)) {
    const dim3 g(dtf_cdiv(a.M, 256) * dtf_cdiv(a.N, 256), splits);
    if (planes) hipLaunchKernelGGL((gemm_pp_kernel<EPI + EPI_PLANES, VxGemm>), g, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((gemm_pp_kernel<EPI, VxGemm>), g, dim3(512), 0, s, a);
  } else {
    const dim3 g(dtf_cdiv(a.M, 128) * dtf_cdiv(a.N, 128), splits);
    if (planes) hipLaunchKernelGGL((gemm_tiled_kernel<unsigned short, EPI + EPI_PLANES, 4, 4, VxGemm>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((gemm_tiled_kernel<unsigned short, EPI, 4, 4, VxGemm>), g, dim3(256), 0, s, a);
  }
}

template <int EPI>
void launch_skinny_f32(const VxGemm& a, hipStream_t s) {
  const dim3 g((unsigned)(dtf_cdiv(a.M, 16) * dtf_cdiv(a.N, 64)));
  const bool aligned = a.K % 4 == 0 && a.lda % 4 == 0 && a.ldb % 4 == 0 && dtf_aligned16(a.A) && dtf_aligned16(a.B);
  if (aligned) hipLaunchKernelGGL((vx_skinny_kernel<unsigned int, EPI, true>), g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((vx_skinny_kernel<unsigned int, EPI, false>), g, dim3(256), 0, s, a);
}
template <int EPI>
void launch_skinny(const VxGemm& a, hipStream_t s) {
  if (a.dtype == TK_BF16) {
    hipLaunchKernelGGL((vx_skinny_kernel<unsigned short, EPI, true>), dim3((unsigned)(dtf_cdiv(a.M, 16) * dtf_cdiv(a.N, 64))), dim3(256), 0, s, a);
    return;
  }
  const int rt = skinny_tiles(a.dtype, a.M, a.N);
  const dim3 g((unsigned)(dtf_cdiv(a.M, 16 * rt) * dtf_cdiv(a.N, 64)));
  if (rt == 4) hipLaunchKernelGGL((vx_split_logits_kernel<EPI, 4>), g, dim3(256), 0, s, a);
  else if (rt == 2) hipLaunchKernelGGL((vx_split_logits_kernel<EPI, 2>), g, dim3(256), 0, s, a);
  else launch_skinny_f32<EPI>(a, s);
}

template <int EPI>
void launch_logits(const VxGemm& a, bool skinny, hipStream_t s) {
  if (skinny) launch_skinny<EPI>(a, s);
  else launch_gemm<EPI>(a, 1, s);
}

// planes: 3 bf16 planes an operand, each dense; 1: the operands are of type dtype
VxGemm operands(const void* A, const void* B, int dtype, int planes, int M, int N, int K, long lda, long ldb) {
  VxGemm g = {};
  const long es = planes == 3 || dtype == TK_BF16 ? 2 : 4;
  g.A = A; g.B = B; g.M = M; g.N = N; g.K = K;
  g.lda = (int)lda; g.ldb = (int)ldb; g.dtype = dtype;
  if (planes == 3) {
    g.a_plane = (unsigned)(M * lda * es);
    g.b_plane = (unsigned)(N * ldb * es);
  }
  g.a_bytes = 2 * g.a_plane + (unsigned)(((M - 1) * lda + K) * es);
  g.b_bytes = 2 * g.b_plane + (unsigned)(((N - 1) * ldb + K) * es);
  return g;
}

// How many K ranges a product is cut into, so that its blocks fill the chip: 256x256 blocks (one a CU) if they do with
// ranges of 1024 or more, else 128x128 blocks (two a CU), at least 512 deep.  Planes make every range six times as deep.
int splits_for(int planes, long m, long n, long k) {
  const long deep = planes == 3 ? 128 : 512;
  if (m >= 256 && n >= 256) {
    const long big = ((m + 255) / 256) * ((n + 255) / 256), s = std::max<long>(1, 256 / big);
    if (big * s >= 192 && k / s >= std::max<long>(256, 2 * deep)) return (int)s;
  }
  const long blocks = ((m + 127) / 128) * ((n + 127) / 128);
  return (int)std::max<long>(1, std::min<long>({512 / blocks, k / deep, 32}));
}
long kper_for(long k, int splits) { return up((k + splits - 1) / splits, 128); }

// Sizes of one call: the padded width, the vocabulary piece and the workspace's parts
struct VxPlan {
  // Dp, Np: width and token count padded to 16 bytes (the products' sizes).  Copies' rows are ld* apart, a multiple of 128
  // bytes: rows that straddle cache lines cost twice the requests (dX at 4093 x 50001 x 1024: 432 us with rows of 50008)
  long Dp, Np, Vp, pieces, strips, blocks, ldd, ldn, ldv;
  int K;                                         // of the logits: padded only where both operands are
  int planes;                                    // of every operand of the large products
  bool skinny, direct, small, pack_x, pack_w, direct_dx, direct_dw;       // direct: the logits read X and W (or padded copies) as they are
  int rt;                                        // of few rows: tiles of 16 rows a workgroup of dX
  int sx, sw;                                    // splits of the two products
  size_t x, w, part, target, blk, rows, xt, wt, dz32, dz, dzt, dx32, dw32, db, total;
};

size_t take(size_t& at, size_t bytes) {
  const size_t here = at;
  at += (bytes + 255) & ~(size_t)255;
  return here;
}

VxPlan plan(const DtfVocabXentArgs& a, bool backward) {
  VxPlan p = {};
  const long es = a.dtype == TK_BF16 ? 2 : 4;
  p.planes = a.dtype == TK_BF16 ? 1 : 3;
  p.Dp = up(a.D, 8);
  p.Np = up(a.N, 8);
  p.ldd = up(a.D, 64);
  p.ldn = up(a.N, 64);
  // a piece: dz and its transpose in 1 GiB, but never under 16384 columns (the products' K and M); every operand of a
  // launch stays below 2 GiB (32-bit offsets), and a launch of 128x128 blocks below 2^32 threads
  const long col = 2 * p.planes;                 // bytes an element of an operand takes
  long vp = backward ? std::max<long>((1l << 30) / (2 * col * p.ldn), 16384) : (1l << 30);
  vp = std::min(vp, ((1l << 31) - (1 << 20)) / (col * std::max({p.ldd, (long)a.ldw, backward ? p.ldn : 0})));
  vp = std::min(vp, (1l << 37) / p.ldn);
  vp = std::max<long>(vp / 256 * 256, 256);
  p.pieces = (a.V + vp - 1) / vp;
  p.Vp = p.pieces == 1 ? a.V : std::min(vp, up((a.V + p.pieces - 1) / p.pieces, 256));
  p.pieces = (a.V + p.Vp - 1) / p.Vp;
  p.ldv = up(p.Vp, 64);
  p.skinny = use_skinny(a.dtype, a.N, p.Vp, a.D);
  p.direct = !use_planes(a.dtype, p.skinny);
  p.small = few_rows(a.dtype, a.N);
  // copies: planes, or bf16 rows that are no whole aligned 16-byte pieces
  const bool bf16 = a.dtype == TK_BF16;
  const bool odd_x = a.D % 8 || a.ldx % 8 || !dtf_aligned16(a.X), odd_w = a.D % 8 || a.ldw % 8 || !dtf_aligned16(a.W);
  p.K = p.direct && (!bf16 || a.D % 8 == 0) ? a.D : (int)p.Dp;
  p.pack_x = !p.direct || (bf16 && odd_x);
  p.pack_w = !p.direct || (bf16 && (odd_w || a.w_dtype != a.dtype));
  const size_t copy = p.direct ? es : 6;
  size_t at = 0;
  if (p.pack_x) p.x = take(at, (size_t)a.N * p.ldd * copy);
  if (p.pack_w) p.w = take(at, (size_t)p.Vp * p.ldd * copy);
  if (!backward) {
    p.strips = (a.V + kStrip - 1) / kStrip;
    p.blocks = (a.N + 63) / 64;
    p.part = take(at, (size_t)p.strips * a.N * 8);
    p.target = take(at, (size_t)a.N * 8);
    p.blk = take(at, (size_t)p.blocks * 12);
  } else {
    const long Vpp = up(p.Vp, 8);
    p.rows = take(at, (size_t)up(a.N, 256) * sizeof(VxRow) + 16);     // and the common factor behind them
    if (p.small) {
      p.dz32 = take(at, (size_t)a.N * p.ldv * 4);
      // column tiles x row tiles x ranges of the vocabulary: about 1024 workgroups, ranges of 256 or more
      const int cols = a.w_dtype == TK_BF16 ? 128 : 64;
      const long tiles = (a.D + cols - 1) / cols, ranges = std::max<long>(1, std::min<long>(p.Vp / 256, 256));
      p.rt = row_tiles(a.w_dtype, a.N, tiles * ranges);
      p.sx = (int)std::max<long>(1, std::min<long>(1024 / (tiles * ((a.N + 16 * p.rt - 1) / (16 * p.rt))), ranges));
      p.dx32 = take(at, (size_t)p.pieces * p.sx * a.N * p.Dp * 4);
    } else {
      p.xt = take(at, (size_t)p.Dp * p.ldn * col);
      p.wt = take(at, (size_t)p.Dp * p.ldv * col);
      p.dz = take(at, (size_t)a.N * p.ldv * col);
      p.dzt = take(at, (size_t)p.Vp * p.ldn * col);
      p.sx = splits_for(p.planes, a.N, p.Dp, Vpp);
      p.sw = splits_for(p.planes, p.Vp, p.Dp, p.Np);
      p.sx = (int)((Vpp + kper_for(Vpp, p.sx) - 1) / kper_for(Vpp, p.sx));
      p.sw = (int)((p.Np + kper_for(p.Np, p.sw) - 1) / kper_for(p.Np, p.sw));
      // straight into the result where one product (or the last piece's) holds the whole sum at a 16-byte row width
      p.direct_dx = p.sx == 1 && p.Dp == a.D && dtf_aligned16(a.dX);
      p.direct_dw = p.sw == 1 && p.Dp == a.D && dtf_aligned16(a.dW);
      if (!p.direct_dx || (a.dtype == TK_BF16 && p.pieces > 1)) p.dx32 = take(at, (size_t)p.sx * a.N * p.Dp * 4);
      if (!p.direct_dw) p.dw32 = take(at, (size_t)p.sw * p.Vp * p.Dp * 4);
    }
    if (a.dbias) p.db = take(at, (size_t)(a.N / 16 + 4) * p.Vp * 4);       // one row of partial sums for every 16 rows at most
  }
  p.total = at;
  return p;
}

template <typename T>
void finish_as(const float* ws, int splits, long rows, int cols, int ldw, void* out, long ldo, const float* scale, const VxRow* own, hipStream_t s) {
  const long n = rows * ((cols + 3) / 4);
  hipLaunchKernelGGL((vx_finish_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, ws, splits, (int)rows, cols, ldw, static_cast<T*>(out), ldo, scale, own);
}
void finish(const float* ws, int splits, long rows, int cols, int ldw, void* out, long ldo, int dtype, const float* scale, const VxRow* own, hipStream_t s) {
  if (dtype == TK_BF16) finish_as<unsigned short>(ws, splits, rows, cols, ldw, out, ldo, scale, own, s);
  else finish_as<float>(ws, splits, rows, cols, ldw, out, ldo, scale, own, s);
}

template <typename TS, typename TD>
void pack_as(const void* src, void* dst, long rows, int cols, long lds_, long ldd, hipStream_t s) {
  hipLaunchKernelGGL((vx_pack_kernel<TS, TD>), dim3((unsigned)((rows * ldd + 255) / 256)), dim3(256), 0, s, static_cast<const TS*>(src),
                     static_cast<TD*>(dst), (int)rows, cols, lds_, (int)ldd);
}
void pack(const void* src, int sdt, void* dst, long rows, int cols, long lds_, long ldd, hipStream_t s) {
  if (sdt == TK_F32) pack_as<float, unsigned short>(src, dst, rows, cols, lds_, ldd, s);
  else pack_as<unsigned short, unsigned short>(src, dst, rows, cols, lds_, ldd, s);
}

void transpose(const void* src, void* dst, long M, long N, long lds_, long ldt, const VxRow* rows, bool weighted, hipStream_t s) {
  const dim3 g((unsigned)(((N + 63) / 64) * ((ldt + 63) / 64)));            // one index: there may be more than 65535 tile rows
  hipLaunchKernelGGL(vx_transpose_kernel, g, dim3(256), 0, s, static_cast<const unsigned short*>(src), static_cast<unsigned short*>(dst), (int)M, (int)N, lds_, (int)ldt, rows, (int)weighted);
}

VxPlanes planes_of(const void* src, void* dst, void* dst_t, long M, long N, long lds_, long Np, long Nt, long Mp, const VxRow* rows) {
  return {static_cast<const float*>(src), static_cast<unsigned short*>(dst), static_cast<unsigned short*>(dst_t), rows, lds_, (int)M, (int)N, (int)Np, (int)Nt, (int)Mp,
          (int)(((Np + 63) / 64) * ((Mp + 63) / 64))};
}
// and leaves them empty
void launch_planes(VxPlanes& a, VxPlanes& b, hipStream_t s) {
  if (a.blocks + b.blocks) hipLaunchKernelGGL(vx_planes_kernel, dim3((unsigned)(a.blocks + b.blocks)), dim3(256), 0, s, a, b);
  a.blocks = b.blocks = 0;
}

// One operand of the logits ([rows, D] of `from`, ld apart) as the kernel reads it, and transposed for a product (bf16: from
// the aligned copy; to_t null: not needed).  Planes are left to the caller to launch.
struct Operand { const void* p; long ld; };
Operand prepare(const DtfVocabXentArgs& a, const VxPlan& p, const void* src, int from, long rows, long ld, bool copy, void* dst, void* to_t, long ldt,
                const VxRow* row_info, VxPlanes& planes, hipStream_t s) {
  Operand o = {src, ld};
  if (!p.direct || (p.planes == 3 && to_t)) planes = planes_of(src, p.direct ? nullptr : dst, to_t, rows, a.D, ld, p.ldd, p.Dp, ldt ? ldt : up(rows, 8), row_info);
  if (p.direct && copy) pack(src, from, dst, rows, a.D, ld, p.ldd, s);
  if (copy) o = {dst, p.ldd};
  if (p.planes == 1 && to_t) transpose(o.p, to_t, rows, p.Dp, o.ld, ldt, row_info, row_info && a.dloss_rows, s);
  return o;
}

// fp32 logits that are made of planes, cut beforehand or in registers
void operands_as_they_are(VxGemm& g, const DtfVocabXentArgs& a, long v0, const VxPlan& p) {
  if (a.dtype != TK_F32 || (p.skinny && skinny_tiles(a.dtype, g.M, g.N) == 1)) return;
  g.x32 = static_cast<const float*>(a.X);
  g.w32 = static_cast<const float*>(a.W) + v0 * a.ldw;
  g.ldx32 = a.ldx;
  g.ldw32 = a.ldw;
  g.D = a.D;
}

// dz in fp32 for the kernels of few rows
void launch_small_dz(const VxGemm& a, bool skinny, hipStream_t s) {
  if (skinny) launch_skinny<VX_DZ32>(a, s);
  else hipLaunchKernelGGL((gemm_tiled_kernel<unsigned short, VX_DZ32, 4, 4, VxGemm>), dim3(dtf_cdiv(a.M, 128) * dtf_cdiv(a.N, 128)), dim3(256), 0, s, a);
}

template <typename T, bool ROUND, int RT>
void small_dx_as(const DtfVocabXentArgs& a, const VxPlan& p, const float* dz, long lddz, const void* w, long n, float* out, hipStream_t s) {
  const dim3 g((unsigned)dtf_cdiv(a.D, 256 / (int)sizeof(T)), (unsigned)dtf_cdiv(a.N, 16 * RT), (unsigned)p.sx);
  const int per = (int)up((p.Vp + p.sx - 1) / p.sx, 64);
  hipLaunchKernelGGL((vx_small_dx_kernel<T, ROUND, RT>), g, dim3(256), 0, s, dz, lddz, static_cast<const T*>(w), (long)a.ldw, out, a.N, a.D, n, per, (int)p.Dp);
}
void small_dx(const DtfVocabXentArgs& a, const VxPlan& p, const float* dz, long lddz, const void* w, long n, float* out, hipStream_t s) {
  if (a.w_dtype == TK_BF16) return small_dx_as<unsigned short, false, 1>(a, p, dz, lddz, w, n, out, s);
  if (a.dtype == TK_BF16) return p.rt == 1 ? small_dx_as<float, true, 1>(a, p, dz, lddz, w, n, out, s) : small_dx_as<float, true, 2>(a, p, dz, lddz, w, n, out, s);
  if (p.rt == 1) return small_dx_as<float, false, 1>(a, p, dz, lddz, w, n, out, s);
  const dim3 g((unsigned)dtf_cdiv(a.D, 64), (unsigned)dtf_cdiv(a.N, 16 * p.rt), (unsigned)p.sx);
  const int per = (int)up((p.Vp + p.sx - 1) / p.sx, 64);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, dim3(256), 0, s, dz, lddz, static_cast<const float*>(w), (long)a.ldw, out, a.N, a.D, n, per, (int)p.Dp); };
  if (p.rt == 4) go(vx_split_dx_kernel<4>);
  else go(vx_split_dx_kernel<2>);
}

// Waves of 4 (bf16: 2) tiles of 16 vocabulary rows where two workgroups a CU are left, else of one.  One tile / this, at 65536 x
// 4096, forward and backward: fp32 64 rows 1.51 / 1.43 ms, bf16 32 rows 0.70 / 0.66.
template <typename TX, typename TO, int RT>
void small_dw_as(const DtfVocabXentArgs& a, const float* dz, long lddz, long n, void* out, const VxRow* rows, const float* scale, hipStream_t s) {
  const long blocks = ((n + 64 * RT - 1) / (64 * RT)) * dtf_cdiv(a.D, 256 / (int)sizeof(TX));
  if (RT > 1 && blocks < 512) return small_dw_as<TX, TO, 1>(a, dz, lddz, n, out, rows, scale, s);
  hipLaunchKernelGGL((vx_small_dw_kernel<TX, TO, RT>), dim3((unsigned)blocks), dim3(256), 0, s, dz, lddz, static_cast<const TX*>(a.X), (long)a.ldx,
                     static_cast<TO*>(out), a.N, a.D, n, rows, scale);
}
void small_dw(const DtfVocabXentArgs& a, const float* dz, long lddz, long n, void* out, const VxRow* rows, const float* scale, hipStream_t s) {
  const long blocks = ((n + 255) / 256) * dtf_cdiv(a.D, 64);              // (split_dw below 9 rows: half of its products are with rows that do not exist)
  if (a.dtype == TK_F32 && a.N > 8 && blocks >= 512)
    hipLaunchKernelGGL(vx_split_dw_kernel, dim3((unsigned)blocks), dim3(256), 0, s, dz, lddz, static_cast<const float*>(a.X), (long)a.ldx, static_cast<float*>(out), a.N, a.D,
                       n, rows, scale);
  else if (a.dtype == TK_F32) small_dw_as<float, float, 4>(a, dz, lddz, n, out, rows, scale, s);
  else if (a.w_dtype == TK_F32) small_dw_as<unsigned short, float, 2>(a, dz, lddz, n, out, rows, scale, s);
  else small_dw_as<unsigned short, unsigned short, 2>(a, dz, lddz, n, out, rows, scale, s);
}

int check(const DtfVocabXentArgs* a) {
  if (!a) return DTF_ERR_ARG;
  if ((a->dtype != TK_F32 && a->dtype != TK_BF16) || (a->w_dtype != TK_F32 && a->w_dtype != TK_BF16)) return DTF_ERR_ARG;
  if (a->w_dtype == TK_BF16 && a->dtype == TK_F32) return DTF_ERR_ARG;
  if (a->N <= 0 || a->V <= 0 || a->D <= 0 || a->ldx < a->D || a->ldw < a->D) return DTF_ERR_SHAPE;
  const long es = a->dtype == TK_BF16 ? 2 : 6, limit = (1l << 31) - (1 << 20);          // fp32: three bf16 planes
  if (a->V > (1l << 30) || a->N > (1l << 26) || a->D > (1l << 20)) return DTF_ERR_SHAPE;
  if (a->N * std::max<long>(a->ldx, up(a->D, 64)) * es > limit || up(a->D, 64) * 256 * es > limit || up(a->N, 64) * 256 * es > limit) return DTF_ERR_SHAPE;
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
  if (!a.X || !a.W || !a.labels || !a.lse || !a.top || !a.total || !a.loss_rows || !a.loss || !a.counts || !a.ws) return DTF_ERR_ARG;
  const VxPlan p = plan(a, false);
  if (a.ws_bytes < (int64_t)p.total) return DTF_ERR_SHAPE;
  if (!dtf_aligned16(a.ws)) return DTF_ERR_ALIGN;
  char* const ws = static_cast<char*>(a.ws);
  VxPlanes of_x = {}, of_w = {};
  const Operand X = prepare(a, p, a.X, a.dtype, a.N, a.ldx, p.pack_x, ws + p.x, nullptr, 0, nullptr, of_x, s);
  const int large = p.direct ? 1 : p.planes;     // planes of the logits' operands
  for (long v0 = 0; v0 < a.V; v0 += p.Vp) {
    const long n = std::min<long>(p.Vp, a.V - v0);
    const Operand W = prepare(a, p, static_cast<const char*>(a.W) + v0 * a.ldw * (a.w_dtype == TK_BF16 ? 2 : 4), a.w_dtype, n, a.ldw, p.pack_w, ws + p.w, nullptr, 0, nullptr, of_w, s);
    launch_planes(of_x, of_w, s);
    VxGemm g = operands(X.p, W.p, a.dtype, large, a.N, (int)n, p.K, X.ld, W.ld);
    g.bias = a.bias ? a.bias + v0 : nullptr;
    g.labels = a.labels;
    g.part = reinterpret_cast<float2*>(ws + p.part);
    g.target = reinterpret_cast<float2*>(ws + p.target);
    g.v0 = (int)v0;
    operands_as_they_are(g, a, v0, p);
    launch_logits<VX_LSE>(g, p.skinny, s);
  }
  VxJoin j = {reinterpret_cast<const float2*>(ws + p.part), reinterpret_cast<const float2*>(ws + p.target), a.labels, a.lse, a.top, a.total, a.loss_rows, a.loss,
              a.counts, reinterpret_cast<float*>(ws + p.blk), reinterpret_cast<int*>(ws + p.blk + p.blocks * 4), a.N, (int)p.strips, (int)p.blocks,
              a.mean, a.V, a.ignore};
  hipLaunchKernelGGL(vx_join_kernel, dim3((unsigned)p.blocks), dim3(64 * kLseSplits), 0, s, j);
  if (p.blocks > 1) hipLaunchKernelGGL(vx_total_kernel, dim3(1), dim3(256), 0, s, j);
  return dtf_check_launch();
}

DTF_EXPORT int dtf_vocab_xent_bwd(const DtfVocabXentArgs* ap, hipStream_t s) {
  if (const int rc = check(ap)) return rc;
  const DtfVocabXentArgs& a = *ap;
  if (!a.X || !a.W || !a.labels || !a.top || !a.total || !a.counts || !a.ws || !(a.dX || a.dW || a.dbias)) return DTF_ERR_ARG;
  const VxPlan p = plan(a, true);
  if (a.ws_bytes < (int64_t)p.total) return DTF_ERR_SHAPE;
  if (!dtf_aligned16(a.ws)) return DTF_ERR_ALIGN;
  char* const ws = static_cast<char*>(a.ws);
  VxRow* const rows = reinterpret_cast<VxRow*>(ws + p.rows);
  const int Mp = (int)up(a.N, 256);
  float* const scale = reinterpret_cast<float*>(rows + Mp);
  const bool apart = p.planes == 1 && !p.small;  // dz is rounded to bf16
  const VxRow* const own = apart && a.dloss_rows ? rows : nullptr;
  if (own) hipLaunchKernelGGL(vx_largest_kernel, dim3(1), dim3(1024), 0, s, a.dloss, a.labels, a.N, a.V, a.ignore, scale);
  hipLaunchKernelGGL(vx_rows_kernel, dim3(Mp / 256), dim3(256), 0, s, a.top, a.total, a.labels, a.dloss, a.dloss_rows, a.counts, a.mean, a.N, Mp, a.V, a.ignore, (int)apart,
                     rows, scale);
  VxPlanes of_x = {}, of_w = {};
  const Operand X = prepare(a, p, a.X, a.dtype, a.N, a.ldx, p.pack_x, ws + p.x, a.dW && !p.small ? ws + p.xt : nullptr, p.ldn, rows, of_x, s);
  const int large = p.direct ? 1 : p.planes;     // planes of the logits' operands
  float* const dx32 = reinterpret_cast<float*>(ws + p.dx32);
  float* const dw32 = reinterpret_cast<float*>(ws + p.dw32);
  for (long v0 = 0; v0 < a.V; v0 += p.Vp) {
    const long n = std::min<long>(p.Vp, a.V - v0), np = up(n, 8), ldv = up(n, 64);
    const Operand W = prepare(a, p, static_cast<const char*>(a.W) + v0 * a.ldw * (a.w_dtype == TK_BF16 ? 2 : 4), a.w_dtype, n, a.ldw, p.pack_w, ws + p.w,
                              a.dX && !p.small ? ws + p.wt : nullptr, ldv, nullptr, of_w, s);
    launch_planes(of_x, of_w, s);
    VxGemm g = operands(X.p, W.p, a.dtype, large, a.N, (int)n, p.K, X.ld, W.ld);
    g.bias = a.bias ? a.bias + v0 : nullptr;
    operands_as_they_are(g, a, v0, p);
    g.rows = rows;
    g.v0 = (int)v0;
    g.C = p.small ? ws + p.dz32 : a.dX ? ws + p.dz : nullptr;
    g.ldc = (int)ldv;
    g.Ct = a.dW && !p.small ? ws + p.dzt : nullptr;
    g.ldct = (int)p.ldn;
    g.db_part = a.dbias ? reinterpret_cast<float*>(ws + p.db) : nullptr;
    if (p.small) launch_small_dz(g, p.skinny, s);
    else launch_logits<VX_DZ>(g, p.skinny, s);
    if (a.dbias)
      hipLaunchKernelGGL(vx_db_kernel, dim3(dtf_cdiv((int)n, 256)), dim3(256), 0, s, g.db_part, dtf_cdiv(a.N, wave_rows(g, p.skinny)), (int)n, a.dbias + v0, scale);
    if (p.small) {
      const float* const dz = reinterpret_cast<const float*>(ws + p.dz32);
      if (a.dX) small_dx(a, p, dz, ldv, static_cast<const char*>(a.W) + v0 * a.ldw * (a.w_dtype == TK_BF16 ? 2 : 4), n, dx32 + (size_t)(v0 / p.Vp) * p.sx * a.N * p.Dp, s);
      if (a.dW) small_dw(a, dz, ldv, n, static_cast<char*>(a.dW) + v0 * a.D * (a.w_dtype == TK_BF16 ? 2 : 4), rows, scale, s);
      continue;
    }
    if (a.dX) {
      VxGemm d = operands(ws + p.dz, ws + p.wt, TK_BF16, p.planes, a.N, (int)p.Dp, (int)np, ldv, ldv);
      const long kper = kper_for(up(p.Vp, 8), p.sx);
      const int splits = (int)((np + kper - 1) / kper);
      d.kper = p.sx > 1 ? (int)kper : 0;
      d.C32 = p.direct_dx && a.dtype == TK_F32 ? static_cast<float*>(a.dX) : dx32;
      d.ldc32 = (int)p.Dp;
      d.accumulate = v0 > 0;                     // the last, shorter piece adds to its first splits only
      if (p.direct_dx && v0 + n == a.V) {
        d.scale = scale;
        d.rows = own;
        if (a.dtype == TK_BF16) d.C = a.dX;
        d.ldc = a.D;
      }
      launch_gemm<VX_SUM>(d, splits, s);
    }
    if (a.dW) {
      VxGemm d = operands(ws + p.dzt, ws + p.xt, TK_BF16, p.planes, (int)n, (int)p.Dp, (int)p.Np, p.ldn, p.ldn);
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
      if (!p.direct_dw) finish(dw32, p.sw, n, a.D, (int)p.Dp, out, a.D, a.w_dtype, scale, nullptr, s);
    }
  }
  if (a.dX && !p.direct_dx) finish(dx32, p.small ? (int)p.pieces * p.sx : p.sx, a.N, a.D, (int)p.Dp, a.dX, a.D, a.dtype, scale, own, s);
  return dtf_check_launch();
}
