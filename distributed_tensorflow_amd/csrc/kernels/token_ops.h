// Shared pieces of the token-model kernels (layernorm.hip, dropout.hip, embedding.hip, vocab_xent.hip): element types,
// 16-byte loads and stores of bf16 / fp32 rows, wave reductions, the counter-based generator.
#pragma once
#include "dtf_common.h"

typedef unsigned int tk_u32x4 __attribute__((ext_vector_type(4)));

enum { TK_F32 = 0, TK_BF16 = 1 };          // dtype codes of the C ABI (the same as the tiled GEMM's)

__device__ __forceinline__ float tk_bf2f(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ unsigned short tk_f2bf(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }   // nearest even
__device__ __forceinline__ unsigned tk_pack2(float a, float b) { return (unsigned)tk_f2bf(a) | ((unsigned)tk_f2bf(b) << 16); }

// One element, whatever its type: unsigned short carries bf16 bits.
__device__ __forceinline__ float tk_get(const unsigned short* p) { return tk_bf2f(*p); }
__device__ __forceinline__ float tk_get(const float* p) { return *p; }
__device__ __forceinline__ void tk_put(unsigned short* p, float v) { *p = tk_f2bf(v); }
__device__ __forceinline__ void tk_put(float* p, float v) { *p = v; }
// The value an element has after it has been stored (what a later reader sees).
__device__ __forceinline__ float tk_round(const unsigned short*, float v) { return tk_bf2f(tk_f2bf(v)); }
__device__ __forceinline__ float tk_round(const float*, float v) { return v; }

// VEC elements: 8 bf16 or 4 fp32 are one 16-byte access (p 16-byte aligned), 1 is an element.
template <typename T, int VEC> struct TkVec;
template <> struct TkVec<unsigned short, 8> {
  static __device__ __forceinline__ void unpack(const tk_u32x4& q, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(q[i] << 16);
      v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ tk_u32x4 pack(const float (&v)[8]) {
    return tk_u32x4{tk_pack2(v[0], v[1]), tk_pack2(v[2], v[3]), tk_pack2(v[4], v[5]), tk_pack2(v[6], v[7])};
  }
  static __device__ __forceinline__ void load(const unsigned short* p, float (&v)[8]) { unpack(*reinterpret_cast<const tk_u32x4*>(p), v); }
  static __device__ __forceinline__ void store(unsigned short* p, const float (&v)[8]) { *reinterpret_cast<tk_u32x4*>(p) = pack(v); }
};
template <> struct TkVec<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const f32x4 q = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q[i];
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) { *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]}; }
};
// A row piece of VEC elements at column c of a row of C, as the 16 bytes that a lane holds: ALIGNED where every piece is
// whole and 16-byte aligned, else by one 16-byte access at the elements' own alignment (the hardware splits it where it
// crosses a line) and element by element in the row's last piece.
typedef tk_u32x4 tk_u32x4_at2 __attribute__((aligned(2)));
template <typename T, bool ALIGNED>
struct TkPiece {
  static constexpr int VEC = 16 / sizeof(T);
  static __device__ __forceinline__ tk_u32x4 load(const T* row, int c, int C) {
    if (ALIGNED) return *reinterpret_cast<const tk_u32x4*>(row + c);
    if (c + VEC <= C) return *reinterpret_cast<const tk_u32x4_at2*>(row + c);
    tk_u32x4 q = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < VEC - 1; ++i)
      if (c + i < C) {
        if (sizeof(T) == 4) q[i] = __builtin_bit_cast(unsigned, tk_get(reinterpret_cast<const float*>(row) + c + i));
        else q[i >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(row)[c + i] << (16 * (i & 1));
      }
    return q;
  }
  static __device__ __forceinline__ void unpack(const tk_u32x4& q, float (&v)[VEC]) {
    if constexpr (sizeof(T) == 2) {
      TkVec<unsigned short, 8>::unpack(q, v);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(q[i]);
    }
  }
  static __device__ __forceinline__ void store(T* row, int c, int C, const float (&v)[VEC]) {
    tk_u32x4 q;
    if constexpr (sizeof(T) == 2) q = TkVec<unsigned short, 8>::pack(v);
    else q = __builtin_bit_cast(tk_u32x4, f32x4{v[0], v[1], v[2], v[3]});
    if (ALIGNED) {
      *reinterpret_cast<tk_u32x4*>(row + c) = q;
    } else if (c + VEC <= C) {
      *reinterpret_cast<tk_u32x4_at2*>(row + c) = q;
    } else {
#pragma unroll
      for (int i = 0; i < VEC - 1; ++i)
        if (c + i < C) tk_put(row + c + i, v[i]);
    }
  }
};

template <typename T> struct TkVec<T, 1> {
  static __device__ __forceinline__ void load(const T* p, float (&v)[1]) { v[0] = tk_get(p); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[1]) { tk_put(p, v[0]); }
};

// VEC elements at c of a parameter vector (weight, bias) of C elements and either type (a wave-uniform flag), by 16-byte
// accesses at the elements' own alignment; `rest` past its end.
typedef f32x4 tk_f32x4_at4 __attribute__((aligned(4)));
template <int VEC>
__device__ __forceinline__ void tk_load_param(const void* p, int bf16, int c, int C, float rest, float (&v)[VEC]) {
  if (VEC >= 4 && c + VEC <= C) {
    if (bf16) {
      const unsigned short* const q = static_cast<const unsigned short*>(p) + c;
      if constexpr (VEC == 8) {
        const tk_u32x4 piece = *reinterpret_cast<const tk_u32x4_at2*>(q);
        TkVec<unsigned short, 8>::unpack(piece, v);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = tk_bf2f(q[i]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC / 4; ++k) {
        const f32x4 q = *reinterpret_cast<const tk_f32x4_at4*>(static_cast<const float*>(p) + c + 4 * k);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * k + i] = q[i];
      }
    }
  } else if (bf16) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = c + i < C ? tk_bf2f(static_cast<const unsigned short*>(p)[c + i]) : rest;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = c + i < C ? static_cast<const float*>(p)[c + i] : rest;
  }
}

// Every lane ends with the sum over the wave.
__device__ __forceinline__ float tk_wave_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, false));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x122, 0xf, 0xf, false));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x121, 0xf, 0xf, false));
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): four random words for a 128-bit counter under a 64-bit key.
__device__ __forceinline__ void tk_philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[1] = (uint32_t)p1; c[3] = (uint32_t)p0;
    c[0] = n0; c[2] = n2;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
}
