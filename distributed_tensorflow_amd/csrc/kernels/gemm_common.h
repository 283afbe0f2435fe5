// What the two tiled GEMM kernels (gemm_pingpong.h, gemm_tiled.h) share: raw buffer access, element types, epilogues.
#pragma once
#include "dtf_kernels.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
static constexpr unsigned kOOB = 0xFFFFFFF0u;

// EPI_WGRAD_OPT: weight gradient with the optimizer folded in (8-wave kernel).  From EPI_CUSTOM on the epilogue belongs
// to the argument struct: p.select() chooses the operands' K range and the tile before the main loop, p.epilogue<EPI>(...)
// takes the accumulators after it (vocab_xent.hip).
// With EPI_PLANES added, A and B are three bf16 planes each whose sum is the fp32 operand (p.a_plane, p.b_plane bytes
// apart), and the product is the sum of the six plane products of 2^-16 and more (gemm_plane_pair): the K loop runs over the
// pairs one after the other.
enum { EPI_FWD = 0, EPI_BWD = 1, EPI_WGRAD = 2, EPI_WGRAD_OPT = 3, EPI_CUSTOM = 4, EPI_PLANES = 32 };

// K-tile kt of a product of planes with nk K-tiles a plane: which pair (>= 6: past the last), which tile inside it, where
// the pair's planes start.  Pairs (a, b): 00 01 10 02 20 11.
struct GemmPlaneTile { int pair, tile; unsigned a_off, b_off; };
__device__ __forceinline__ GemmPlaneTile gemm_plane_pair(int kt, int nk, unsigned a_plane, unsigned b_plane) {
  const int pair = (kt >= nk) + (kt >= 2 * nk) + (kt >= 3 * nk) + (kt >= 4 * nk) + (kt >= 5 * nk) + (kt >= 6 * nk);
  return {pair, kt - pair * nk, ((0x120100u >> (4 * pair)) & 3u) * a_plane, ((0x102010u >> (4 * pair)) & 3u) * b_plane};
}
