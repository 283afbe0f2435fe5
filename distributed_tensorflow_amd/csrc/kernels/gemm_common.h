// What the two tiled GEMM kernels (gemm_pingpong.h, gemm_tiled.h) share: raw buffer access, element types, epilogues.
#pragma once
#include "dtf_kernels.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
static constexpr unsigned kOOB = 0xFFFFFFF0u;

// EPI_WGRAD_OPT: weight gradient with the optimizer folded in (8-wave kernel).  From EPI_CUSTOM on the epilogue belongs
// to the argument struct: p.select(blockIdx.y) before the main loop, p.epilogue<EPI>(...) after it (vocab_xent.hip).
enum { EPI_FWD = 0, EPI_BWD = 1, EPI_WGRAD = 2, EPI_WGRAD_OPT = 3, EPI_CUSTOM = 4 };
