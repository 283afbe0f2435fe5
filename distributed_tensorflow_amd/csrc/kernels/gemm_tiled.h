// The kernel of gemm_tiled.hip, as a template that other files can give an epilogue of their own.
//
// Throughput GEMM for the wide layers:  C[M,N] = A[M,K] . B[N,K]^T   (both operands k-contiguous)
//
// All three products of a dense layer are brought to this one form by keeping
// transposed copies where a product needs them (they are written by the
// producing kernel's epilogue, never by a separate transpose pass over HBM):
//
//   forward    Y  = X  . W        A = X [batch,in]      B = W^T [out,in]      (+bias, ReLU)
//   backward   dX = dY . W^T      A = dY [batch,out]    B = W   [in,out]      (* (act > 0))
//   gradient   dW = X^T . dY      A = X^T [in,batch]    B = dY^T [out,batch]  (+ db = rowsum(dY^T))
//
// This file: the register-staged 4-wave kernels, which take every shape (ragged edges through the range check of
// the buffer loads) and both dtypes; large aligned bf16 products go to the 8-wave kernel in gemm_pingpong.hip
// (dispatch in launch_tiled below).
// Tile: 128x128 per workgroup, 4 waves (2x2), each wave 64x64 = 4x4 MFMA tiles of 16x16 (or 256x256 with 8x8
// tiles per wave, see the template parameters).
// K-step per LDS stage: 128 bytes per row (64 bf16 / 32 fp32), two stages (double buffer),
// register-staged: the global loads of stage t+1 are issued before the MFMAs of stage t and
// written to the other LDS buffer after them, one barrier per stage.
// LDS rows are 128 B; the 16-byte slot index is XOR-ed with (row & 7), which makes every
// ds_read_b128 fragment read conflict-free (the 16-lane groups of a b128 read cover 16
// distinct slots of the 256-byte bank row).
// bf16: v_mfma_f32_16x16x32_bf16, fp32 accumulate.  fp32: v_mfma_f32_16x16x4_f32 (exact fp32).
// Workgroup ids are remapped so that the workgroups sharing an XCD (ids equal mod 8) cover a
// contiguous band of tiles and share operand panels in that XCD's L2.
#pragma once
#include "gemm_common.h"

__device__ __forceinline__ rsrc_t make_rsrc(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ unsigned short f2bf(float f) {  // round to nearest even; NaN stays NaN
  return __builtin_bit_cast(unsigned short, (__bf16)f);
}
__device__ __forceinline__ float bf2f(unsigned short h) { return __uint_as_float((unsigned)h << 16); }

template <typename T> struct Elem;
template <> struct Elem<unsigned short> { static constexpr int PER16 = 8; };   // bf16 elements per 16 bytes
template <> struct Elem<unsigned int> { static constexpr int PER16 = 4; };      // fp32 carried as its bit pattern

template <typename T>
__device__ __forceinline__ void mma_slot(const u32x4& a, const u32x4& b, f32x4& c);
template <>
__device__ __forceinline__ void mma_slot<unsigned short>(const u32x4& a, const u32x4& b, f32x4& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ void mma_slot<unsigned int>(const u32x4& a, const u32x4& b, f32x4& c) {
  // lane group g holds k = 4g..4g+3 of this 16-deep slot; MFMA j consumes element j of every group
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
}

// TI x TJ: MFMA tiles per wave (wave tile 16*TI x 16*TJ); the 2x2 waves of a workgroup cover 32*TI x 32*TJ.
//   4 x 4: 128x128 block, 64 KB of LDS, two workgroups per CU; per 16 MFMAs a wave reads 8 fragments, which
//          keeps the LDS port saturated (measured: the loop is LDS-read bound).
//   8 x 8: 256x256 block, 128 KB of LDS, one workgroup per CU; 16 fragment reads per 64 MFMAs halve the LDS
//          traffic per flop.  Used for bf16 when the problem fills the chip with such blocks.
template <typename T, int EPI, int TI, int TJ, class Args>
__global__ __launch_bounds__(256) void gemm_tiled_kernel(Args p) {
  constexpr int PER16 = Elem<T>::PER16;
  constexpr int BKE = 8 * PER16;             // elements per 128-byte LDS row
  constexpr int BM = 32 * TI, BN = 32 * TJ;
  __shared__ __attribute__((aligned(16))) unsigned char lds_a[2][BM * 128];   // [stage][row*128 + byte]
  __shared__ __attribute__((aligned(16))) unsigned char lds_b[2][BN * 128];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;

  const int tiles_n = (p.N + BN - 1) / BN, tiles_m = (p.M + BM - 1) / BM;
  int wg;
  if constexpr (EPI >= EPI_CUSTOM) wg = p.select();
  else wg = dtf_xcd_remap(blockIdx.x, tiles_m * tiles_n);
  // consecutive (remapped) ids walk down a column band of 8 row-tiles: A panels and one B panel stay in L2
  const int band = 8;
  const int per_band = band * tiles_n;
  const int b_idx = wg / per_band, in_band = wg % per_band;
  const int rows_in_band = min(band, tiles_m - b_idx * band);
  const int tm = b_idx * band + in_band % rows_in_band;
  const int tn = in_band / rows_in_band;
  const int m0 = tm * BM, n0 = tn * BN;

  const rsrc_t ra = make_rsrc(p.A, p.a_bytes), rb = make_rsrc(p.B, p.b_bytes);

  // staging map: BM*8 (A) and BN*8 (B) 16-byte chunks per stage, TI resp. TJ per thread; chunk = (row, slot)
  unsigned a_goff[TI], b_goff[TJ];
  unsigned la_off[TI], lb_off[TJ];
#pragma unroll
  for (int c = 0; c < TI; ++c) {
    const int id = tid + 256 * c;
    const int row = id >> 3, slot = id & 7;
    a_goff[c] = (m0 + row < p.M) ? (unsigned)(m0 + row) * (unsigned)p.lda * (unsigned)sizeof(T) + (unsigned)slot * 16u : kOOB;
    la_off[c] = (unsigned)row * 128u + (unsigned)((slot ^ (row & 7)) << 4);
  }
#pragma unroll
  for (int c = 0; c < TJ; ++c) {
    const int id = tid + 256 * c;
    const int row = id >> 3, slot = id & 7;
    b_goff[c] = (n0 + row < p.N) ? (unsigned)(n0 + row) * (unsigned)p.ldb * (unsigned)sizeof(T) + (unsigned)slot * 16u : kOOB;
    lb_off[c] = (unsigned)row * 128u + (unsigned)((slot ^ (row & 7)) << 4);
  }
  const int nstage_plane = (p.K + BKE - 1) / BKE;
  const int nstage = EPI >= EPI_PLANES ? 6 * nstage_plane : nstage_plane;
  const int my_slot = tid & 7;               // (tid + 256 c) & 7 for every c
  u32x4 ra_reg[TI], rb_reg[TJ];
  auto stage_load = [&](int t) {
    int k0 = t * BKE;
    unsigned ka = 0, kb = 0;
    if constexpr (EPI >= EPI_PLANES) {
      const GemmPlaneTile q = gemm_plane_pair(t, nstage_plane, p.a_plane, p.b_plane);
      k0 = q.tile * BKE;
      ka = q.a_off;
      kb = q.b_off;
    }
    const bool kin = k0 + my_slot * PER16 < p.K;           // K is a multiple of PER16 (checked by the launcher)
    ka += (unsigned)k0 * (unsigned)sizeof(T);
    kb += (unsigned)k0 * (unsigned)sizeof(T);
#pragma unroll
    for (int c = 0; c < TI; ++c)
      ra_reg[c] = __builtin_amdgcn_raw_buffer_load_b128(ra, (int)((kin && a_goff[c] != kOOB) ? a_goff[c] + ka : kOOB), 0, 0);
#pragma unroll
    for (int c = 0; c < TJ; ++c)
      rb_reg[c] = __builtin_amdgcn_raw_buffer_load_b128(rb, (int)((kin && b_goff[c] != kOOB) ? b_goff[c] + kb : kOOB), 0, 0);
  };
  auto stage_write = [&](int buf) {
#pragma unroll
    for (int c = 0; c < TI; ++c) *reinterpret_cast<u32x4*>(&lds_a[buf][la_off[c]]) = ra_reg[c];
#pragma unroll
    for (int c = 0; c < TJ; ++c) *reinterpret_cast<u32x4*>(&lds_b[buf][lb_off[c]]) = rb_reg[c];
  };

  f32x4 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float bias_grad[TJ];
#pragma unroll
  for (int j = 0; j < TJ; ++j) bias_grad[j] = 0.f;

  // fragment read offsets: row r = wave base + 16 i + fr, slot s = 4 ks + g  ->  r*128 + ((s ^ (r & 7)) << 4)
  const unsigned a_rbase = (unsigned)(wm * 16 * TI + fr) * 128u, b_rbase = (unsigned)(wn * 16 * TJ + fr) * 128u;
  const int sw = fr & 7;     // (row & 7) == (fr & 7): the row bases are multiples of 16

  auto read_frags = [&](int buf, int ks, u32x4 (&af)[TI], u32x4 (&bf)[TJ]) {
    const unsigned so = (unsigned)(((4 * ks + g) ^ sw) << 4);
#pragma unroll
    for (int j = 0; j < TJ; ++j) bf[j] = *reinterpret_cast<const u32x4*>(&lds_b[buf][b_rbase + (unsigned)j * 2048u + so]);
#pragma unroll
    for (int i = 0; i < TI; ++i) af[i] = *reinterpret_cast<const u32x4*>(&lds_a[buf][a_rbase + (unsigned)i * 2048u + so]);
  };
  auto bias_accumulate = [&](const u32x4 (&bf)[TJ]) {
    // db[n] = sum_k dY^T[n][k]: each lane adds the 16 bytes it holds of its B rows
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      if (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias_grad[j] += bf2f((unsigned short)(bf[j][e] & 0xffff)) + bf2f((unsigned short)(bf[j][e] >> 16));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias_grad[j] += __uint_as_float(bf[j][e]);
      }
    }
  };

  stage_load(0);
  stage_write(0);
  __syncthreads();
  if (TI >= 8) {
    // One wave per SIMD: nothing else hides an LDS read, so the fragments of the second k-step are requested
    // before the MFMAs of the first (two fragment sets in registers), and the next stage's operands are
    // written to the other buffer between the two k-steps.
    u32x4 af0[TI], bf0[TJ], af1[TI], bf1[TJ];
    for (int t = 0; t < nstage; ++t) {
      const int cur = t & 1;
      const bool more = t + 1 < nstage;
      if (more) stage_load(t + 1);
      read_frags(cur, 0, af0, bf0);
      read_frags(cur, 1, af1, bf1);
      __builtin_amdgcn_sched_barrier(0);
      if (EPI == EPI_WGRAD) bias_accumulate(bf0);
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) mma_slot<T>(af0[i], bf0[j], acc[i][j]);
      if (more) stage_write(cur ^ 1);          // last read a barrier ago
      if (EPI == EPI_WGRAD) bias_accumulate(bf1);
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) mma_slot<T>(af1[i], bf1[j], acc[i][j]);
      __syncthreads();
    }
  } else {
    for (int t = 0; t < nstage; ++t) {
      const int cur = t & 1;
      if (t + 1 < nstage) stage_load(t + 1);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x4 af[TI], bf[TJ];
        read_frags(cur, ks, af, bf);
        if (EPI == EPI_WGRAD) bias_accumulate(bf);
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
          for (int j = 0; j < TJ; ++j) mma_slot<T>(af[i], bf[j], acc[i][j]);
      }
      if (t + 1 < nstage) stage_write(cur ^ 1);
      __syncthreads();
    }
  }

  if constexpr (EPI >= EPI_CUSTOM) {       // the barrier that ends the main loop leaves the staging buffers free
    static_assert(TI == 4 && TJ == 4, "one 16 KB piece of the staging buffers for each wave's 64x64 block");
    unsigned char* const wl = (wave < 2 ? lds_a[wave] : lds_b[wave - 2]);
    p.template epilogue<EPI & ~EPI_PLANES, (EPI >= EPI_PLANES || sizeof(T) == 4)>(acc, wl, m0 + wm * 64, n0 + wn * 64, lane);
    return;
  }
  // ---------------- epilogue: acc[i][j][r] = C[m0 + wm*16*TI + 16i + 4g + r][n0 + wn*16*TJ + 16j + fr]
  T* __restrict__ C = static_cast<T*>(p.C);
  T* __restrict__ Ct = static_cast<T*>(p.Ct);
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    const int col = n0 + wn * 16 * TJ + 16 * j + fr;
    const bool col_ok = col < p.N;
    const float bias = (EPI == EPI_FWD && p.bias && col_ok) ? p.bias[col] : 0.f;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int row0 = m0 + wm * 16 * TI + 16 * i + 4 * g;
      float v[4];
      float mk[4] = {1.f, 1.f, 1.f, 1.f};
      if (EPI == EPI_BWD && col_ok) {
        if (p.maskT && row0 + 3 < p.M && (p.ldmaskt & 3) == 0) {
          // the lane's four rows are contiguous in the transposed mask: one load instead of four
          const T* mt = static_cast<const T*>(p.maskT) + (size_t)col * p.ldmaskt + row0;
          if (sizeof(T) == 2) {
            const uint2 q = *reinterpret_cast<const uint2*>(mt);
            mk[0] = bf2f((unsigned short)(q.x & 0xffff)); mk[1] = bf2f((unsigned short)(q.x >> 16));
            mk[2] = bf2f((unsigned short)(q.y & 0xffff)); mk[3] = bf2f((unsigned short)(q.y >> 16));
          } else {
            const float4 q = *reinterpret_cast<const float4*>(mt);
            mk[0] = q.x; mk[1] = q.y; mk[2] = q.z; mk[3] = q.w;
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (row0 + r < p.M) {
              const T m = static_cast<const T*>(p.mask)[(size_t)(row0 + r) * p.ldmask + col];
              mk[r] = sizeof(T) == 2 ? bf2f((unsigned short)m) : __uint_as_float((unsigned)m);
            }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = acc[i][j][r] + bias;
        if (EPI == EPI_FWD && p.relu) v[r] = fmaxf(v[r], 0.f);
        if (EPI == EPI_BWD) v[r] = mk[r] > 0.f ? v[r] : 0.f;
      }
      if (!col_ok) continue;
      if (EPI == EPI_WGRAD) {
        float* __restrict__ Cf = static_cast<float*>(p.C);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row0 + r < p.M) Cf[(size_t)(row0 + r) * p.ldc + col] = v[r];
        continue;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (row0 + r < p.M) {
          if (sizeof(T) == 2) C[(size_t)(row0 + r) * p.ldc + col] = (T)f2bf(v[r]);
          else C[(size_t)(row0 + r) * p.ldc + col] = (T)__float_as_uint(v[r]);
          if (p.C32) p.C32[(size_t)(row0 + r) * p.ldc32 + col] = v[r];
        }
      }
      if (Ct) {
        // transposed copy: the 4 rows a lane holds are contiguous in Ct's row `col`
        if (row0 + 3 < p.M && (p.ldct & 3) == 0) {
          if (sizeof(T) == 2) {
            uint2 pk;
            pk.x = (unsigned)f2bf(v[0]) | ((unsigned)f2bf(v[1]) << 16);
            pk.y = (unsigned)f2bf(v[2]) | ((unsigned)f2bf(v[3]) << 16);
            *reinterpret_cast<uint2*>(&Ct[(size_t)col * p.ldct + row0]) = pk;
          } else {
            *reinterpret_cast<float4*>(&Ct[(size_t)col * p.ldct + row0]) = make_float4(v[0], v[1], v[2], v[3]);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (row0 + r < p.M) {
              if (sizeof(T) == 2) Ct[(size_t)col * p.ldct + row0 + r] = (T)f2bf(v[r]);
              else Ct[(size_t)col * p.ldct + row0 + r] = (T)__float_as_uint(v[r]);
            }
        }
      }
    }
  }
  if (EPI == EPI_WGRAD && p.bias_out && tm == 0 && wm == 0) {
    // lanes fr of the 4 lane groups hold disjoint k ranges of B row (wn*16*TJ + 16i + fr)
#pragma unroll
    for (int i = 0; i < TJ; ++i) {
      float s = bias_grad[i];
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      const int col = n0 + wn * 16 * TJ + 16 * i + fr;
      if (g == 0 && col < p.N) p.bias_out[col] = s;
    }
  }
}
