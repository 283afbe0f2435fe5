// Layer normalisation over the last axis: forward (optionally of x + residual) and backward with the reduction of the
// weight's and bias's gradients.
//
//   h = x [+ residual], stored in x's type;  mean = sum h / C;  var = sum (h - mean)^2 / C;  rstd = 1 / sqrt(var + eps)
//   xhat = (h - mean) rstd;  y = xhat w + b
//   g = dy w;  dx = rstd (g - sum g / C - xhat sum(g xhat) / C) [+ dh];  dw = sum_rows dy xhat;  db = sum_rows dy
//
// All sums are fp32.  The variance is the sum of squared distances from the mean (two reductions over registers): the
// sum of squares minus the squared mean would cancel for rows whose mean is large against their spread.
//
// Layout.  A row belongs to TPR threads (one wave up to a whole workgroup) and is read ONCE into registers with 16-byte
// accesses (8 bf16 / 4 fp32; at the elements' own alignment where width, stride or address ask for it).  TPR is the smallest
// of 64 / 256 / 512 / 1024 for which a thread holds at most 16 elements (backward: 32 past 8192 columns): in the backward
// pass a thread keeps its columns' running dw and db, the weight, xhat and g in registers, five floats an element.  The
// backward pass runs on at most 256 workgroups of 512 threads, each walking over rows and leaving ONE partial [dw | db] (so
// the partials stay a few per cent of the traffic); while a row's sums cross the workgroup, the next row is already on its
// way: 8 waves a CU with 96 bytes a lane in flight cover the latency at full bandwidth.  A second launch adds the partials
// in workgroup order.  No atomics: the same inputs give the same bits.  Bound by memory: 8192 x 4096 bf16 with residual
// takes 51 us forward and 55 + 6 us backward, 268 MB each: 5.3 and 4.9 TB/s (a 4 GiB copy: 4.75).  Rows too wide for registers are streamed
// (three passes forward, two backward, column sums on their own).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "token_ops.h"

namespace {
constexpr int kBlock = 1024;
constexpr int kBwdBlock = 512;               // 256 registers a thread: the backward pass keeps a row, its gradients and the next row
constexpr int kMaxParts = 256;               // workgroups of the backward pass, one per CU

struct LnArgs {
  const void* x; const void* res; const void* w; const void* b; void* y; void* h; float* mean; float* rstd;
  long rows; int C; long ldx, ldres; int w_bf16; float eps;
};
struct LnBwdArgs {
  const void* dy; const void* h; const void* dh; const void* w; const float* mean; const float* rstd; void* dx; float* part;
  long rows; int C; long lddy, ldh, lddh; int w_bf16, want_wgrad;
};

// Sums of one or two values over the TPR threads of a row; `s` holds one float a wave and value, in two alternating
// halves, so that one barrier a call suffices (a wave can only reach the call after next, which writes the same half
// again, once every wave has read this one).
template <int TPR, int NVAL>
__device__ __forceinline__ void row_sum(float (&v)[NVAL], float (*s)[NVAL][kBlock / 64], int& half) {
#pragma unroll
  for (int k = 0; k < NVAL; ++k) v[k] = tk_wave_sum(v[k]);
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6, first = wave & ~(TPR / 64 - 1);
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < NVAL; ++k) s[half][k][wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NVAL; ++k) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 64; ++i) t += s[half][k][first + i];
      v[k] = t;
    }
    half ^= 1;
  }
}

template <typename T, bool AL, int NV, int TPR, int BLOCK>
__global__ __launch_bounds__(BLOCK) void ln_fwd_kernel(LnArgs a) {
  typedef TkPiece<T, AL> P;
  constexpr int VEC = P::VEC;
  __shared__ float s_sum[2][1][kBlock / 64];
  const int t = threadIdx.x % TPR;
  const long row = ((long)blockIdx.y * gridDim.x + blockIdx.x) * (BLOCK / TPR) + threadIdx.x / TPR;
  const bool live = row < a.rows;            // dead rows of the last workgroup still take part in its barriers
  const T* const x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ldx;
  tk_u32x4 raw[NV];
  float v[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * VEC;
    raw[j] = live && c < a.C ? P::load(x, c, a.C) : tk_u32x4{0u, 0u, 0u, 0u};
  }
  if (a.res) {
    const T* const r = static_cast<const T*>(a.res) + (live ? row : 0) * a.ldres;
    T* const h = static_cast<T*>(a.h) + row * a.C;
    tk_u32x4 rr[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * VEC;
      rr[j] = live && c < a.C ? P::load(r, c, a.C) : tk_u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * VEC;
      float q[VEC];
      P::unpack(raw[j], v[j]);
      P::unpack(rr[j], q);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = tk_round(h, v[j][i] + q[i]);         // normalised as the stream stores it
      if (live && c < a.C) P::store(h, c, a.C, v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) P::unpack(raw[j], v[j]);
  }
  float w[NV][VEC], b[NV][VEC];                // asked for before the sums, needed after them
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) { w[j][i] = 1.f; b[j][i] = 0.f; }
    if (a.w && c < a.C) tk_load_param<VEC>(a.w, a.w_bf16, c, AL ? 0x7fffffff : a.C, 1.f, w[j]);
    if (a.b && c < a.C) tk_load_param<VEC>(a.b, a.w_bf16, c, AL ? 0x7fffffff : a.C, 0.f, b[j]);
  }
  int half = 0;
  float s[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[0] += v[j][i];           // zeros past the row's end
  row_sum<TPR, 1>(s, s_sum, half);
  const float inv_c = 1.f / (float)a.C;
  const float mean = s[0] * inv_c;
  s[0] = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[j][i] -= mean;
      if (AL ? c < a.C : c + i < a.C) s[0] = fmaf(v[j][i], v[j][i], s[0]);
    }
  }
  row_sum<TPR, 1>(s, s_sum, half);
  const float rstd = 1.f / sqrtf(s[0] * inv_c + a.eps);
  if (!live) return;
  if (t == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  T* const y = static_cast<T*>(a.y) + row * a.C;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * VEC;
    if (c < a.C) {
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = fmaf(v[j][i] * rstd, w[j][i], b[j][i]);
      P::store(y, c, a.C, o);
    }
  }
}

// Rows too wide for registers: the row is read three times (twice from L2).
template <typename T>
__global__ __launch_bounds__(kBlock) void ln_fwd_stream_kernel(LnArgs a) {
  __shared__ float s_sum[2][1][kBlock / 64];
  const long row = (long)blockIdx.y * gridDim.x + blockIdx.x;
  if (row >= a.rows) return;
  const T* src = static_cast<const T*>(a.x) + row * a.ldx;
  const T* const r = a.res ? static_cast<const T*>(a.res) + row * a.ldres : nullptr;
  T* const h = a.res ? static_cast<T*>(a.h) + row * a.C : nullptr;
  int half = 0;
  float s[1] = {0.f};
  for (int c = threadIdx.x; c < a.C; c += kBlock) {
    float v = tk_get(src + c);
    if (r) {
      v = tk_round(h, v + tk_get(r + c));
      tk_put(h + c, v);                      // read back below by the thread that wrote it
    }
    s[0] += v;
  }
  if (r) src = h;
  row_sum<kBlock, 1>(s, s_sum, half);
  const float inv_c = 1.f / (float)a.C, mean = s[0] * inv_c;
  s[0] = 0.f;
  for (int c = threadIdx.x; c < a.C; c += kBlock) {
    const float d = tk_get(src + c) - mean;
    s[0] = fmaf(d, d, s[0]);
  }
  row_sum<kBlock, 1>(s, s_sum, half);
  const float rstd = 1.f / sqrtf(s[0] * inv_c + a.eps);
  if (threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  T* const y = static_cast<T*>(a.y) + row * a.C;
  for (int c = threadIdx.x; c < a.C; c += kBlock) {
    float w[1] = {1.f}, b[1] = {0.f};
    if (a.w) tk_load_param<1>(a.w, a.w_bf16, c, a.C, 1.f, w);
    if (a.b) tk_load_param<1>(a.b, a.w_bf16, c, a.C, 0.f, b);
    tk_put(y + c, fmaf((tk_get(src + c) - mean) * rstd, w[0], b[0]));
  }
}

template <typename T, bool AL, int NV, int TPR>
__global__ __launch_bounds__(kBwdBlock) void ln_bwd_kernel(LnBwdArgs a) {
  typedef TkPiece<T, AL> P;
  constexpr int VEC = P::VEC, RPB = kBwdBlock / TPR, COLS = NV * TPR * VEC;
  constexpr bool AHEAD = NV * VEC <= 16;     // the next row's pieces fit the registers
  __shared__ float s_sum[2][2][kBlock / 64];
  __shared__ float s_col[RPB > 1 ? COLS : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float w[NV][VEC], aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) { w[j][i] = 1.f; aw[j][i] = 0.f; ab[j][i] = 0.f; }
    if (a.w && c < a.C) tk_load_param<VEC>(a.w, a.w_bf16, c, AL ? 0x7fffffff : a.C, 0.f, w[j]);
  }
  const float inv_c = 1.f / (float)a.C;
  int half = 0;
  const long step = (long)gridDim.x * RPB;
  // what a row brings: dy and h as loaded, its statistics; zeros past the row's end and for rows that do not exist
  tk_u32x4 ndy[NV], nh[NV];
  float nmean, nrstd;
  auto fetch = [&](long row) {
    const bool live = row < a.rows;
    const T* const dy = static_cast<const T*>(a.dy) + (live ? row : 0) * a.lddy;
    const T* const h = static_cast<const T*>(a.h) + (live ? row : 0) * a.ldh;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * VEC;
      const bool in = live && c < a.C;
      nh[j] = in ? P::load(h, c, a.C) : tk_u32x4{0u, 0u, 0u, 0u};
      ndy[j] = in ? P::load(dy, c, a.C) : tk_u32x4{0u, 0u, 0u, 0u};
    }
    nmean = live ? a.mean[row] : 0.f;
    nrstd = live ? a.rstd[row] : 0.f;
  };
  if (AHEAD) fetch((long)blockIdx.x * RPB + sub);
  for (long row0 = (long)blockIdx.x * RPB; row0 < a.rows; row0 += step) {      // the same count for every wave
    const long row = row0 + sub;
    const bool live = row < a.rows;
    if (!AHEAD) fetch(row);
    const float mean = nmean, rstd = nrstd;
    float xh[NV][VEC], g[NV][VEC];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * VEC;
      P::unpack(nh[j], xh[j]);
      P::unpack(ndy[j], g[j]);                 // dy = 0 past the row's end: no share in any sum, whatever xh is there
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        xh[j][i] = (xh[j][i] - mean) * rstd;
        if (!AL && c + i >= a.C) xh[j][i] = 0.f;
        aw[j][i] = fmaf(g[j][i], xh[j][i], aw[j][i]);
        ab[j][i] += g[j][i];
        g[j][i] *= w[j][i];
        s[0] += g[j][i];
        s[1] = fmaf(g[j][i], xh[j][i], s[1]);
      }
    }
    if (AHEAD) fetch(row + step);              // on its way while the sums below cross the workgroup
    tk_u32x4 q[NV];
    if (a.dh) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * VEC;
        q[j] = live && c < a.C ? P::load(static_cast<const T*>(a.dh) + row * a.lddh, c, a.C) : tk_u32x4{0u, 0u, 0u, 0u};
      }
    }
    row_sum<TPR, 2>(s, s_sum, half);
    const float m1 = s[0] * inv_c, m2 = s[1] * inv_c;
    if (live) {
      T* const dx = static_cast<T*>(a.dx) + row * a.C;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * VEC;
        if (c < a.C) {
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = rstd * (g[j][i] - fmaf(xh[j][i], m2, m1));
          if (a.dh) {
            float z[VEC];
            P::unpack(q[j], z);
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] += z[i];
          }
          P::store(dx, c, a.C, o);
        }
      }
    }
  }
  if (!a.want_wgrad) return;
  // this workgroup's partial: the subgroups add into LDS in their order, the last one stores
  float* const part = a.part + (size_t)blockIdx.x * 2 * a.C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    for (int k = 0; k < RPB; ++k) {
      if (RPB > 1) __syncthreads();
      if (sub == k) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int c = (j * TPR + t) * VEC + i;
            float v = which ? ab[j][i] : aw[j][i];
            if (RPB > 1 && k > 0) v += s_col[c];
            if (RPB > 1 && k < RPB - 1) s_col[c] = v;
            else if (c < a.C) part[(size_t)which * a.C + c] = v;
          }
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void ln_bwd_stream_kernel(LnBwdArgs a) {
  __shared__ float s_sum[2][2][kBlock / 64];
  const long row = (long)blockIdx.y * gridDim.x + blockIdx.x;
  if (row >= a.rows) return;
  const T* const dy = static_cast<const T*>(a.dy) + row * a.lddy;
  const T* const h = static_cast<const T*>(a.h) + row * a.ldh;
  const T* const dh = a.dh ? static_cast<const T*>(a.dh) + row * a.lddh : nullptr;
  T* const dx = static_cast<T*>(a.dx) + row * a.C;
  const float mean = a.mean[row], rstd = a.rstd[row], inv_c = 1.f / (float)a.C;
  int half = 0;
  float s[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < a.C; c += kBlock) {
    float w[1] = {1.f};
    if (a.w) tk_load_param<1>(a.w, a.w_bf16, c, a.C, 1.f, w);
    const float g = tk_get(dy + c) * w[0];
    s[0] += g;
    s[1] = fmaf(g, (tk_get(h + c) - mean) * rstd, s[1]);
  }
  row_sum<kBlock, 2>(s, s_sum, half);
  const float m1 = s[0] * inv_c, m2 = s[1] * inv_c;
  for (int c = threadIdx.x; c < a.C; c += kBlock) {
    float w[1] = {1.f};
    if (a.w) tk_load_param<1>(a.w, a.w_bf16, c, a.C, 1.f, w);
    float o = rstd * (tk_get(dy + c) * w[0] - fmaf((tk_get(h + c) - mean) * rstd, m2, m1));
    if (dh) o += tk_get(dh + c);
    tk_put(dx + c, o);
  }
}

// Column sums for the streamed rows: workgroup (column tile, row range), one thread a column.
template <typename T>
__global__ __launch_bounds__(256) void ln_colsum_kernel(LnBwdArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  const long per = (a.rows + gridDim.y - 1) / gridDim.y, lo = per * blockIdx.y, hi = min(a.rows, lo + per);
  float sw = 0.f, sb = 0.f;
  for (long row = lo; row < hi; ++row) {
    const float dy = tk_get(static_cast<const T*>(a.dy) + row * a.lddy + c);
    sw = fmaf(dy, (tk_get(static_cast<const T*>(a.h) + row * a.ldh + c) - a.mean[row]) * a.rstd[row], sw);
    sb += dy;
  }
  float* const part = a.part + (size_t)blockIdx.y * 2 * a.C;
  part[c] = sw;
  part[(size_t)a.C + c] = sb;
}

// dw[c], db[c] = the partials' sums: 16 threads a column take every 16th partial each, joined in a fixed order.
__global__ __launch_bounds__(1024) void ln_join_kernel(const float* __restrict__ part, int nparts, int C, void* dw, void* db, int bf16) {
  __shared__ float s[16][65];
  const int lane = threadIdx.x & 63, k = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float v = 0.f;
  if (c < C)
    for (int p = k; p < nparts; p += 16) v += part[((size_t)p * 2 + blockIdx.y) * C + c];
  s[k][lane] = v;
  __syncthreads();
  if (k == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 16; ++i) v += s[i][lane];
    void* const out = blockIdx.y ? db : dw;
    if (!out) return;
    if (bf16) static_cast<unsigned short*>(out)[c] = tk_f2bf(v);
    else static_cast<float*>(out)[c] = v;
  }
}

bool vec_ok(const void* p, long ld, int vec, int es) { return !p || (((uintptr_t)p & 15) == 0 && ld % vec == 0 && vec * es == 16); }

// `blocks` workgroups as a grid of two indices: a launch's x may not reach 2^32 threads
dim3 grid2(long blocks) {
  const long x = std::min<long>(blocks, 1 << 20);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

template <typename T, bool AL, int NV, int TPR>
void fwd_as(const LnArgs& a, hipStream_t s) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  const long rpb = BLOCK / TPR;
  hipLaunchKernelGGL((ln_fwd_kernel<T, AL, NV, TPR, BLOCK>), grid2((a.rows + rpb - 1) / rpb), dim3(BLOCK), 0, s, a);
}

template <typename T, bool AL>
void fwd_width(const LnArgs& a, hipStream_t s) {
  constexpr int VEC = TkPiece<T, AL>::VEC, N16 = 16 / VEC;              // N16 pieces a thread: 16 elements
  if (a.C <= 64 * VEC) fwd_as<T, AL, 1, 64>(a, s);
  else if (a.C <= 64 * 16) fwd_as<T, AL, N16, 64>(a, s);
  else if (a.C <= 256 * 16) fwd_as<T, AL, N16, 256>(a, s);
  else if (a.C <= 512 * 16) fwd_as<T, AL, N16, 512>(a, s);
  else if (a.C <= 1024 * 16) fwd_as<T, AL, N16, 1024>(a, s);
  else hipLaunchKernelGGL((ln_fwd_stream_kernel<T>), grid2(a.rows), dim3(kBlock), 0, s, a);
}

int bwd_parts(long rows, int C) {
  if (C > 1024 * 16) return (int)std::min<long>(std::max<long>(1, rows / 64), 64);
  const long rpb = kBwdBlock / (C <= 64 * 16 ? 64 : C <= 256 * 16 ? 256 : 512);
  return (int)std::min<long>((rows + rpb - 1) / rpb, kMaxParts);
}

template <typename T, bool AL>
void bwd_width(const LnBwdArgs& a, int parts, hipStream_t s) {
  constexpr int VEC = TkPiece<T, AL>::VEC, N16 = 16 / VEC;
  const dim3 g(parts), b(kBwdBlock);
  if (a.C <= 64 * VEC) hipLaunchKernelGGL((ln_bwd_kernel<T, AL, 1, 64>), g, b, 0, s, a);
  else if (a.C <= 64 * 16) hipLaunchKernelGGL((ln_bwd_kernel<T, AL, N16, 64>), g, b, 0, s, a);
  else if (a.C <= 256 * 16) hipLaunchKernelGGL((ln_bwd_kernel<T, AL, N16, 256>), g, b, 0, s, a);
  else if (a.C <= 512 * 16) hipLaunchKernelGGL((ln_bwd_kernel<T, AL, N16, 512>), g, b, 0, s, a);
  else if (a.C <= 1024 * 16) hipLaunchKernelGGL((ln_bwd_kernel<T, AL, 2 * N16, 512>), g, b, 0, s, a);
  else {
    hipLaunchKernelGGL((ln_bwd_stream_kernel<T>), grid2(a.rows), dim3(kBlock), 0, s, a);
    if (a.want_wgrad) hipLaunchKernelGGL((ln_colsum_kernel<T>), dim3(dtf_cdiv(a.C, 256), parts), dim3(256), 0, s, a);
  }
}
}  // namespace

// Rows [rows, C] with leading dimensions ldx / ldres; y and h are dense.  res and h: both or neither; w, b: may be null.
DTF_EXPORT int dtf_layernorm_fwd(const void* x, const void* res, const void* w, const void* b, void* y, void* h, float* mean,
                                 float* rstd, int64_t rows, int C, int64_t ldx, int64_t ldres, int dtype, int w_dtype, float eps,
                                 hipStream_t s) {
  if (rows < 0 || C <= 0 || C > (1 << 30) || rows > 0x7fffffffLL || ldx < C || (res && ldres < C)) return DTF_ERR_SHAPE;
  if ((dtype != TK_F32 && dtype != TK_BF16) || (w_dtype != TK_F32 && w_dtype != TK_BF16) || (res == nullptr) != (h == nullptr)) return DTF_ERR_ARG;
  if (rows == 0) return DTF_OK;
  if (!x || !y || !mean || !rstd) return DTF_ERR_ARG;
  const LnArgs a = {x, res, w, b, y, h, mean, rstd, (long)rows, C, (long)ldx, (long)ldres, w_dtype, eps};
  const int es = dtype == TK_BF16 ? 2 : 4, vec = 16 / es;
  const bool v = C % vec == 0 && vec_ok(x, ldx, vec, es) && vec_ok(res, ldres, vec, es) && vec_ok(y, C, vec, es) && vec_ok(h, C, vec, es);
  if (dtype == TK_BF16) v ? fwd_width<unsigned short, true>(a, s) : fwd_width<unsigned short, false>(a, s);
  else v ? fwd_width<float, true>(a, s) : fwd_width<float, false>(a, s);
  return dtf_check_launch();
}

// Floats of the workspace `part` that the backward pass needs.
DTF_EXPORT int64_t dtf_layernorm_bwd_ws_floats(int64_t rows, int C) {
  return rows <= 0 || C <= 0 ? 0 : (int64_t)bwd_parts((long)rows, C) * 2 * C;
}

// dw, db (dtype w_dtype): null to leave one out; part only if one of them is wanted.
DTF_EXPORT int dtf_layernorm_bwd(const void* dy, const void* h, const void* dh, const void* w, const float* mean, const float* rstd,
                                 void* dx, void* dw, void* db, float* part, int64_t rows, int C, int64_t lddy, int64_t ldh,
                                 int64_t lddh, int dtype, int w_dtype, hipStream_t s) {
  if (rows < 0 || C <= 0 || C > (1 << 30) || rows > 0x7fffffffLL || lddy < C || ldh < C || (dh && lddh < C)) return DTF_ERR_SHAPE;
  if ((dtype != TK_F32 && dtype != TK_BF16) || (w_dtype != TK_F32 && w_dtype != TK_BF16)) return DTF_ERR_ARG;
  const bool wgrad = dw || db;
  LnBwdArgs a = {dy, h, dh, w, mean, rstd, dx, part, (long)rows, C, (long)lddy, (long)ldh, (long)lddh, w_dtype, wgrad};
  int parts = 0;
  if (rows > 0) {
    if (!dy || !h || !mean || !rstd || !dx || (wgrad && !part)) return DTF_ERR_ARG;
    parts = bwd_parts((long)rows, C);
    const int es = dtype == TK_BF16 ? 2 : 4, vec = 16 / es;
    const bool v = C % vec == 0 && vec_ok(dy, lddy, vec, es) && vec_ok(h, ldh, vec, es) && vec_ok(dh, lddh, vec, es) && vec_ok(dx, C, vec, es);
    if (dtype == TK_BF16) v ? bwd_width<unsigned short, true>(a, parts, s) : bwd_width<unsigned short, false>(a, parts, s);
    else v ? bwd_width<float, true>(a, parts, s) : bwd_width<float, false>(a, parts, s);
  }
  if (wgrad)
    hipLaunchKernelGGL(ln_join_kernel, dim3(dtf_cdiv(C, 64), 2), dim3(1024), 0, s, part, parts, C, dw, db, w_dtype);
  return dtf_check_launch();
}
