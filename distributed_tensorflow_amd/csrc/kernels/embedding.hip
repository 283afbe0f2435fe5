// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   forward    y[i] = scale table[id_i]                (an id outside the table gives a row of zeros)
//   backward   dtable[v] = scale sum_{i: id_i = v} dy[i]     for every row of the table, zeros where no token has it
//
// The gradient is a segmented sum.  Tokens are sorted by id, stably, so a row's tokens stand in the order of their
// positions; every table row is then written exactly once, as its tokens' sum or as zeros, by the workgroup that owns it:
// no atomics on floats (the same inputs give the same bits), no zero fill beforehand, no fp32 table in between.
//   sort    LSD radix sort of (id, position) with digits of at most 9 bits (32 KB of counters): up to 16384 tokens in ONE workgroup and launch,
//           else count / scan / scatter launches over blocks of 4096 tokens.
//   parts   A row with more than `chunk` tokens would be summed by one workgroup one token after the other: the sorted
//           list is cut into chunks, and each chunk's share of such a row is summed by a workgroup of its own.
//   rows    32 table rows a workgroup: binary searches in the sorted ids give the rows' tokens, then each row is summed in
//           fp32 (its tokens in order, or the chunks' parts in order), scaled and rounded once.
// Bound by memory: the table's gradient is written once (V D elements), dy is read once.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "token_ops.h"

namespace {
constexpr int kOne = 16384;                      // tokens that one workgroup sorts
constexpr int kSortBlock = 1024, kSortWaves = kSortBlock / 64;
constexpr int kKeys = 4096;                      // tokens a workgroup of the multi-launch sort
constexpr int kMaxBits = 9, kMaxDigits = 1 << kMaxBits;
constexpr int kRows = 32;                        // table rows a workgroup of the last launch

// ---------------------------------------------------------------------------------------------------------- forward
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_fwd_kernel(const void* __restrict__ ids, int ids64, const T* __restrict__ table, T* __restrict__ y, long n, long V,
                                                      int D, long ld, float scale, int tpr_log2) {
  const int tpr = 1 << tpr_log2, t = threadIdx.x & (tpr - 1);
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) >> tpr_log2;
  if (i >= n) return;
  const long id = ids64 ? (long)static_cast<const long long*>(ids)[i] : (long)static_cast<const int*>(ids)[i];
  const bool in = id >= 0 && id < V;
  const T* const src = table + (in ? id : 0) * ld;
  for (int c = t * VEC; c < D; c += tpr * VEC) {
    float v[VEC];
    if (in) {
      TkVec<T, VEC>::load(src + c, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] *= scale;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = 0.f;
    }
    TkVec<T, VEC>::store(y + i * D + c, v);
  }
}

// ------------------------------------------------------------------------------------------------------------- sort
// The key of token i: its id, or V (sorted behind every row, never read again) for tokens without a gradient.
__device__ __forceinline__ int key_of(const void* ids, int ids64, long i, long V, long long skip) {
  const long long id = ids64 ? static_cast<const long long*>(ids)[i] : (long long)static_cast<const int*>(ids)[i];
  return id < 0 || id >= V || id == skip ? (int)V : (int)id;
}

struct SortArgs {
  const void* ids; const int* key_in; const int* pos_in; int* key_out; int* pos_out; int* hist;    // hist [digits][blocks]
  long V; long long skip; int n, ids64, shift, bits, blocks;
};

__device__ __forceinline__ int load_key(const SortArgs& a, int i) { return a.key_in ? a.key_in[i] : key_of(a.ids, a.ids64, i, a.V, a.skip); }

// lanes of the wave whose digit equals this lane's (inactive lanes excluded)
__device__ __forceinline__ unsigned long long same_digit(int digit, int bits, bool active) {
  unsigned long long m = __ballot(active);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long set = __ballot((digit >> b) & 1);
    m &= (digit >> b) & 1 ? set : ~set;
  }
  return m;
}

// One stable pass over the keys [lo, hi) by a workgroup.  cnt [waves][digits] in LDS holds, for every wave, where its next
// key with that digit goes; a wave takes a contiguous range of keys, 64 at a time.
__device__ __forceinline__ void scatter_range(const SortArgs& a, int lo, int hi, int* cnt, int per_wave) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << a.bits, mask = digits - 1;
  int* const mine = cnt + wave * digits;
  const int begin = lo + wave * per_wave, end = min(hi, begin + per_wave);
  for (int base = begin; base < end; base += 64) {
    const int i = base + lane;
    const bool active = i < end;
    const int key = active ? load_key(a, i) : 0, pos = active ? (a.pos_in ? a.pos_in[i] : i) : 0;
    const int digit = (key >> a.shift) & mask;
    const unsigned long long same = same_digit(digit, a.bits, active);
    const int before = (int)__popcll(same & ((1ull << lane) - 1ull));
    if (active) {
      const int at = mine[digit] + before;
      a.key_out[at] = key;
      a.pos_out[at] = pos;
    }
    __builtin_amdgcn_wave_barrier();             // every lane has read its counter before the last of each digit moves it on
    if (active && (same >> lane) == 1ull) mine[digit] += before + 1;
    __builtin_amdgcn_wave_barrier();
  }
}

__device__ __forceinline__ void count_waves(const SortArgs& a, int lo, int hi, int* cnt, int per_wave) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << a.bits;
  for (int i = threadIdx.x; i < kSortWaves * digits; i += kSortBlock) cnt[i] = 0;
  __syncthreads();
  const int begin = lo + wave * per_wave, end = min(hi, begin + per_wave);
  for (int i = begin + lane; i < end; i += 64) atomicAdd(&cnt[wave * digits + ((load_key(a, i) >> a.shift) & (digits - 1))], 1);
  __syncthreads();
}

// Exclusive prefix sum over the workgroup's threads.
__device__ __forceinline__ int block_exclusive(int v, int* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += s_wave[w];
  __syncthreads();
  return before + x - v;
}

// All passes in one workgroup; key/pos buffers a and b alternate, the last pass ends in a.
__global__ __launch_bounds__(kSortBlock) void emb_sort_one_kernel(SortArgs a, int passes, int* key_a, int* pos_a, int* key_b, int* pos_b) {
  extern __shared__ int cnt[];                   // [waves][digits]
  __shared__ int s_wave[kSortWaves];
  const int digits = 1 << a.bits, per_wave = (a.n + kSortBlock - 1) / kSortBlock * 64;
  for (int p = 0; p < passes; ++p) {
    const bool to_a = ((passes - 1 - p) & 1) == 0;
    a.key_in = p == 0 ? nullptr : to_a ? key_b : key_a;
    a.pos_in = p == 0 ? nullptr : to_a ? pos_b : pos_a;
    a.key_out = to_a ? key_a : key_b;
    a.pos_out = to_a ? pos_a : pos_b;
    a.shift = p * a.bits;
    count_waves(a, 0, a.n, cnt, per_wave);
    // totals per digit (one a thread), prefix over the digits, then over the waves
    const int d = threadIdx.x;
    int total = 0;
    if (d < digits)
      for (int w = 0; w < kSortWaves; ++w) total += cnt[w * digits + d];
    int at = block_exclusive(total, s_wave);
    if (d < digits)
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = cnt[w * digits + d];
        cnt[w * digits + d] = at;
        at += c;
      }
    __syncthreads();
    scatter_range(a, 0, a.n, cnt, per_wave);
    __threadfence_block();
    __syncthreads();                             // this pass's keys are written before the next pass reads them
  }
}

__global__ __launch_bounds__(kSortBlock) void emb_count_kernel(SortArgs a) {
  __shared__ int h[kMaxDigits];
  const int digits = 1 << a.bits;
  for (int d = threadIdx.x; d < digits; d += kSortBlock) h[d] = 0;
  __syncthreads();
  const int lo = blockIdx.x * kKeys, hi = min(a.n, lo + kKeys);
  for (int i = lo + threadIdx.x; i < hi; i += kSortBlock) atomicAdd(&h[(load_key(a, i) >> a.shift) & (digits - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortBlock) a.hist[(size_t)d * a.blocks + blockIdx.x] = h[d];
}

// hist: counts -> where each (digit, block) starts
__global__ __launch_bounds__(kSortBlock) void emb_scan_kernel(int* hist, int n) {
  __shared__ int s_wave[kSortWaves];
  const int per = (n + kSortBlock - 1) / kSortBlock, lo = min(n, (int)threadIdx.x * per), hi = min(n, lo + per);
  int sum = 0;
  for (int i = lo; i < hi; ++i) sum += hist[i];
  int at = block_exclusive(sum, s_wave);
  for (int i = lo; i < hi; ++i) {
    const int c = hist[i];
    hist[i] = at;
    at += c;
  }
}

__global__ __launch_bounds__(kSortBlock) void emb_scatter_kernel(SortArgs a) {
  extern __shared__ int cnt[];
  const int digits = 1 << a.bits, lo = blockIdx.x * kKeys, hi = min(a.n, lo + kKeys);
  count_waves(a, lo, hi, cnt, kKeys / kSortWaves);
  for (int d = threadIdx.x; d < digits; d += kSortBlock) {
    int at = a.hist[(size_t)d * a.blocks + blockIdx.x];
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w * digits + d];
      cnt[w * digits + d] = at;
      at += c;
    }
  }
  __syncthreads();
  scatter_range(a, lo, hi, cnt, kKeys / kSortWaves);
}

// ------------------------------------------------------------------------------------------------------------- sums
__device__ __forceinline__ int lower_bound(const int* __restrict__ key, int n, int v) {
  int lo = 0, len = n;
  while (len > 0) {
    const int half = len >> 1;
    if (key[lo + half] < v) { lo += half + 1; len -= half + 1; } else len = half;
  }
  return lo;
}

struct SumArgs {
  const int* key; const int* pos; const void* dy; float* part; void* out;
  long V, lddy; int n, D, chunk, tpr_log2; float scale;
};

template <typename T, int VEC>
__device__ __forceinline__ void add_tokens(const SumArgs& a, int s, int e, int c, float (&acc)[VEC]) {
  const T* const dy = static_cast<const T*>(a.dy);
  for (int i = s; i < e; i += 4) {
    float v[4][VEC];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u < e) TkVec<T, VEC>::load(dy + a.pos[i + u] * a.lddy + c, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u < e) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += v[u][k];
      }
  }
}

// Workgroup (chunk, column tile): the chunk's share of the at most two rows that have more tokens than a chunk holds: the
// one of its first token (part 0) and the one of its last token (part 1, if it is another).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_parts_kernel(SumArgs a) {
  const int lo = blockIdx.x * a.chunk, hi = min(a.n, lo + a.chunk);
  const int c = (blockIdx.y * 256 + threadIdx.x) * VEC;
  const int first = a.key[lo], last = a.key[hi - 1];
  for (int k = 0; k < 2; ++k) {
    const int v = k ? last : first;
    if (v >= a.V || (k && last == first)) continue;
    const bool crosses = (lo > 0 && a.key[lo - 1] == v) || (hi < a.n && a.key[hi] == v);
    if (!crosses) continue;
    const int s = lower_bound(a.key, a.n, v), e = lower_bound(a.key, a.n, v + 1);
    if (e - s <= a.chunk || c >= a.D) continue;
    float acc[VEC] = {};
    add_tokens<T, VEC>(a, max(s, lo), min(e, hi), c, acc);
#pragma unroll
    for (int q = 0; q < VEC; ++q) a.part[((size_t)blockIdx.x * 2 + k) * a.D + c + q] = acc[q];
  }
}

// Workgroup (32 table rows, column tile); 2^tpr_log2 threads a row.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_rows_kernel(SumArgs a) {
  __shared__ int s_at[kRows + 1];
  const long v0 = (long)blockIdx.x * kRows;
  if (threadIdx.x <= kRows) s_at[threadIdx.x] = lower_bound(a.key, a.n, (int)min(v0 + threadIdx.x, a.V));
  __syncthreads();
  const int tpr = 1 << a.tpr_log2, t = threadIdx.x & (tpr - 1);
  const int c = (blockIdx.y * tpr + t) * VEC;
  if (c >= a.D) return;
  T* const out = static_cast<T*>(a.out);
  for (int r = threadIdx.x >> a.tpr_log2; r < kRows; r += 256 >> a.tpr_log2) {
    const long v = v0 + r;
    if (v >= a.V) break;
    const int s = s_at[r], e = s_at[r + 1];
    float acc[VEC] = {};
    if (e - s <= a.chunk) {
      add_tokens<T, VEC>(a, s, e, c, acc);
    } else {
      for (int k = s / a.chunk; k <= (e - 1) / a.chunk; ++k) {
        const int which = s > k * a.chunk;       // not the row of the chunk's first token: of its last
        const float* const p = a.part + ((size_t)k * 2 + which) * a.D + c;
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] += p[q];
      }
    }
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] *= a.scale;
    TkVec<T, VEC>::store(out + v * a.D + c, acc);
  }
}

// --------------------------------------------------------------------------------------------------------- host side
struct EmbPlan {
  int bits, passes, blocks, chunk, chunks;
  size_t key_a, pos_a, key_b, pos_b, hist, part, total;
};

EmbPlan plan(int64_t n, int64_t V, int D) {
  EmbPlan p = {};
  int total = 1;
  while ((1ll << total) <= V) ++total;           // keys 0 .. V
  p.passes = (total + kMaxBits - 1) / kMaxBits;
  p.bits = (total + p.passes - 1) / p.passes;
  p.blocks = (int)((n + kKeys - 1) / kKeys);
  p.chunk = (int)std::min<int64_t>(std::max<int64_t>(64, n / 512), 1024);
  p.chunks = (int)((n + p.chunk - 1) / p.chunk);
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
  p.key_a = take((size_t)n * 4); p.pos_a = take((size_t)n * 4); p.key_b = take((size_t)n * 4); p.pos_b = take((size_t)n * 4);
  p.hist = take(((size_t)p.blocks << p.bits) * 4);
  p.part = take((size_t)p.chunks * 2 * D * 4);
  p.total = at;
  return p;
}

int check(int64_t n, int64_t V, int64_t D, int dtype) {
  if (dtype != TK_F32 && dtype != TK_BF16) return DTF_ERR_ARG;
  if (n < 0 || n > (1ll << 28) || V <= 0 || V > (1ll << 30) || D <= 0 || D > (1 << 20)) return DTF_ERR_SHAPE;
  return DTF_OK;
}

int row_threads_log2(int D, int vec, int most) {
  int l = 0;
  while ((1 << l) * vec < D && (1 << l) < most) ++l;
  return l;
}

template <typename T, int VEC>
void sums(const SumArgs& in, int chunks, hipStream_t s) {
  SumArgs a = in;
  if (a.n > a.chunk)                             // else no row can have more tokens than a chunk
    hipLaunchKernelGGL((emb_parts_kernel<T, VEC>), dim3(chunks, dtf_cdiv(a.D, 256 * VEC)), dim3(256), 0, s, a);
  a.tpr_log2 = row_threads_log2(a.D, VEC, 256);
  hipLaunchKernelGGL((emb_rows_kernel<T, VEC>), dim3((unsigned)((a.V + kRows - 1) / kRows), dtf_cdiv(a.D, VEC << a.tpr_log2)), dim3(256), 0, s, a);
}
}  // namespace

// y [n, D] dense; table rows ldt apart; ids int64 or int32
DTF_EXPORT int dtf_embedding_fwd(const void* ids, int ids64, const void* table, void* y, int64_t n, int64_t V, int D, int64_t ldt, int dtype, float scale,
                                 hipStream_t s) {
  if (const int rc = check(n, V, D, dtype)) return rc;
  if (ldt < D) return DTF_ERR_SHAPE;
  if (n == 0) return DTF_OK;
  if (!ids || !table || !y) return DTF_ERR_ARG;
  const int vec = dtype == TK_BF16 ? 8 : 4;
  const bool v = D % vec == 0 && ldt % vec == 0 && dtf_aligned16(table) && dtf_aligned16(y);
  const int l = row_threads_log2(D, v ? vec : 1, 64);
  const dim3 g((unsigned)(((n << l) + 255) / 256)), b(256);
  if (dtype == TK_BF16) {
    const auto* t = static_cast<const unsigned short*>(table);
    auto* o = static_cast<unsigned short*>(y);
    if (v) hipLaunchKernelGGL((emb_fwd_kernel<unsigned short, 8>), g, b, 0, s, ids, ids64, t, o, (long)n, (long)V, D, (long)ldt, scale, l);
    else hipLaunchKernelGGL((emb_fwd_kernel<unsigned short, 1>), g, b, 0, s, ids, ids64, t, o, (long)n, (long)V, D, (long)ldt, scale, l);
  } else {
    const auto* t = static_cast<const float*>(table);
    auto* o = static_cast<float*>(y);
    if (v) hipLaunchKernelGGL((emb_fwd_kernel<float, 4>), g, b, 0, s, ids, ids64, t, o, (long)n, (long)V, D, (long)ldt, scale, l);
    else hipLaunchKernelGGL((emb_fwd_kernel<float, 1>), g, b, 0, s, ids, ids64, t, o, (long)n, (long)V, D, (long)ldt, scale, l);
  }
  return dtf_check_launch();
}

DTF_EXPORT int64_t dtf_embedding_bwd_ws_bytes(int64_t n, int64_t V, int D) {
  return check(n, V, D, TK_F32) == DTF_OK ? (int64_t)plan(n, V, D).total : -1;
}

// out [V, D] dense of dy's type; tokens whose id is `skip` (or outside the table) give no gradient
DTF_EXPORT int dtf_embedding_bwd(const void* ids, int ids64, const void* dy, void* out, void* ws, int64_t ws_bytes, int64_t n, int64_t V, int D, int64_t lddy,
                                 int dtype, float scale, long long skip, hipStream_t s) {
  if (const int rc = check(n, V, D, dtype)) return rc;
  if (lddy < D) return DTF_ERR_SHAPE;
  if (!out || (n > 0 && (!ids || !dy || !ws))) return DTF_ERR_ARG;
  const EmbPlan p = plan(n, V, D);
  if (n > 0 && ws_bytes < (int64_t)p.total) return DTF_ERR_SHAPE;
  char* const w = static_cast<char*>(ws);
  int* const key_a = reinterpret_cast<int*>(w + p.key_a), * const pos_a = reinterpret_cast<int*>(w + p.pos_a);
  int* const key_b = reinterpret_cast<int*>(w + p.key_b), * const pos_b = reinterpret_cast<int*>(w + p.pos_b);
  SortArgs a = {ids, nullptr, nullptr, nullptr, nullptr, reinterpret_cast<int*>(w + p.hist), (long)V, skip, (int)n, ids64, 0, p.bits, p.blocks};
  const unsigned lds = (unsigned)(kSortWaves << p.bits) * 4u;
  if (n > 0 && n <= kOne) {
    hipLaunchKernelGGL(emb_sort_one_kernel, dim3(1), dim3(kSortBlock), lds, s, a, p.passes, key_a, pos_a, key_b, pos_b);
  } else if (n > 0) {
    for (int k = 0; k < p.passes; ++k) {
      const bool to_a = ((p.passes - 1 - k) & 1) == 0;
      a.key_in = k == 0 ? nullptr : to_a ? key_b : key_a;
      a.pos_in = k == 0 ? nullptr : to_a ? pos_b : pos_a;
      a.key_out = to_a ? key_a : key_b;
      a.pos_out = to_a ? pos_a : pos_b;
      a.shift = k * p.bits;
      hipLaunchKernelGGL(emb_count_kernel, dim3(p.blocks), dim3(kSortBlock), 0, s, a);
      hipLaunchKernelGGL(emb_scan_kernel, dim3(1), dim3(kSortBlock), 0, s, a.hist, p.blocks << p.bits);
      hipLaunchKernelGGL(emb_scatter_kernel, dim3(p.blocks), dim3(kSortBlock), lds, s, a);
    }
  }
  const SumArgs q = {key_a, pos_a, dy, reinterpret_cast<float*>(w + p.part), out, (long)V, (long)lddy, (int)n, D, p.chunk, 0, scale};
  const int vec = dtype == TK_BF16 ? 8 : 4;
  const bool v = D % vec == 0 && lddy % vec == 0 && dtf_aligned16(dy) && dtf_aligned16(out);
  if (dtype == TK_BF16) v ? sums<unsigned short, 8>(q, p.chunks, s) : sums<unsigned short, 1>(q, p.chunks, s);
  else v ? sums<float, 4>(q, p.chunks, s) : sums<float, 1>(q, p.chunks, s);
  return dtf_check_launch();
}
