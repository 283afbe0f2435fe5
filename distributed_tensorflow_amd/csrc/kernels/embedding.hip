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
//   parts   A frequent row summed by one workgroup would take one token after the other: the sorted list is cut into chunks,
//           and each chunk's share of a row that crosses a chunk's border is summed by a workgroup of its own.
//   rows    32 table rows a workgroup: searches in the sorted ids give the rows' tokens, then each row is summed in fp32 (its
//           tokens in order, or the chunks' parts in order), scaled and rounded once.
// Bound by memory: the table's gradient is written once (V D elements), dy is read once.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "token_ops.h"

namespace {
constexpr int kOne = 16384;                      // tokens that one workgroup sorts
constexpr int kSortBlock = 1024, kSortWaves = kSortBlock / 64;
constexpr int kKeys = 4096;                      // tokens a workgroup of the multi-launch sort
constexpr int kMaxBits = 9;
constexpr int kScanBlocks = 256;                 // up to here a scatter block adds up the counts by itself
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
  long V; long long skip; int n, ids64, shift, bits, blocks, scanned;
};

__device__ __forceinline__ int load_key(const SortArgs& a, int i) { return a.key_in ? a.key_in[i] : key_of(a.ids, a.ids64, i, a.V, a.skip); }

// Lanes of the wave whose digit equals this lane's (inactive lanes excluded): one ballot a bit.
__device__ __forceinline__ unsigned long long same_digit(int digit, int bits, bool active) {
  unsigned long long m = __ballot(active);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long set = __ballot((digit >> b) & 1);
    m &= (digit >> b) & 1 ? set : ~set;
  }
  return m;
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

// A wave's keys (ROUNDS x 64 in order, in registers): off[r] = how many earlier keys of the wave have the same digit; after
// the call cnt[wave][digit] holds the wave's count of every digit.  No atomics: the last lane of a digit moves it on.
template <int ROUNDS>
__device__ __forceinline__ void rank_in_wave(const int (&key)[ROUNDS], int live, int shift, int bits, int* mine, int (&off)[ROUNDS]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool active = 64 * r + lane < live;
    const int digit = (key[r] >> shift) & ((1 << bits) - 1);
    const unsigned long long same = same_digit(digit, bits, active);
    const int before = (int)__popcll(same & ((1ull << lane) - 1ull));
    off[r] = active ? mine[digit] + before : 0;
    __builtin_amdgcn_wave_barrier();             // every lane has read its counter before the last of its digit writes it
    if (active && (same >> lane) == 1ull) mine[digit] = off[r] + 1;
    __builtin_amdgcn_wave_barrier();
  }
}

// All passes in one workgroup; keys and positions stay in registers and LDS between them.
__global__ __launch_bounds__(kSortBlock) void emb_sort_one_kernel(SortArgs a, int passes) {
  constexpr int ROUNDS = kOne / kSortBlock;
  __shared__ int s_key[kOne];
  __shared__ unsigned short s_pos[kOne];
  __shared__ int cnt[kSortWaves << kMaxBits];    // [waves][digits]
  __shared__ int s_wave[kSortWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << a.bits;
  const int per_wave = (a.n + kSortBlock - 1) / kSortBlock * 64, lo = wave * per_wave, live = max(0, min(a.n - lo, per_wave));
  int key[ROUNDS], pos[ROUNDS], off[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = lo + 64 * r + lane;
    const bool active = 64 * r + lane < live;
    key[r] = active ? load_key(a, i) : 0;
    pos[r] = i;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * a.bits;
    for (int i = threadIdx.x; i < kSortWaves * digits; i += kSortBlock) cnt[i] = 0;
    __syncthreads();
    rank_in_wave<ROUNDS>(key, live, shift, a.bits, cnt + wave * digits, off);
    __syncthreads();
    // counts -> where each (wave, digit) starts: one digit a thread
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
    const bool last = p == passes - 1;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
      if (64 * r + lane < live) {
        const int to = cnt[wave * digits + ((key[r] >> shift) & (digits - 1))] + off[r];
        if (last) {
          a.key_out[to] = key[r];
          a.pos_out[to] = pos[r];
        } else {
          s_key[to] = key[r];
          s_pos[to] = (unsigned short)pos[r];
        }
      }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
      if (64 * r + lane < live) {
        key[r] = s_key[lo + 64 * r + lane];
        pos[r] = s_pos[lo + 64 * r + lane];
      }
  }
}

__global__ __launch_bounds__(kSortBlock) void emb_count_kernel(SortArgs a) {
  __shared__ int h[1 << kMaxBits];
  const int digits = 1 << a.bits;
  const int lo = blockIdx.x * kKeys, hi = min(a.n, lo + kKeys);
  int key[kKeys / kSortBlock];
#pragma unroll
  for (int r = 0; r < kKeys / kSortBlock; ++r) {
    const int i = lo + r * kSortBlock + threadIdx.x;
    key[r] = i < hi ? load_key(a, i) : -1;
  }
  if ((int)threadIdx.x < digits) h[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kKeys / kSortBlock; ++r)
    if (key[r] >= 0) atomicAdd(&h[(key[r] >> a.shift) & (digits - 1)], 1);     // integers: any order gives the same counts
  __syncthreads();
  if ((int)threadIdx.x < digits) a.hist[(size_t)threadIdx.x * a.blocks + blockIdx.x] = h[threadIdx.x];
}

// hist: counts -> where each (digit, block) starts (more than kScanBlocks blocks: else every scatter block does it itself)
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
  constexpr int ROUNDS = kKeys / kSortBlock;
  __shared__ int cnt[kSortWaves << kMaxBits];
  __shared__ int s_wave[kSortWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << a.bits;
  const int lo = blockIdx.x * kKeys + wave * 64 * ROUNDS, live = max(0, min(a.n - lo, 64 * ROUNDS));
  int key[ROUNDS], pos[ROUNDS], off[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = lo + 64 * r + lane;
    const bool active = 64 * r + lane < live;
    key[r] = active ? load_key(a, i) : 0;
    pos[r] = active && a.pos_in ? a.pos_in[i] : i;
  }
  for (int i = threadIdx.x; i < kSortWaves * digits; i += kSortBlock) cnt[i] = 0;
  // where this block's keys of digit d start: all smaller digits, then the blocks in front
  const int d = threadIdx.x;
  int at = 0;
  if (a.scanned) {
    if (d < digits) at = a.hist[(size_t)d * a.blocks + blockIdx.x];
    __syncthreads();
  } else {
    int total = 0, before = 0;
    if (d < digits)
      for (int b = 0; b < a.blocks; ++b) {
        const int c = a.hist[(size_t)d * a.blocks + b];
        total += c;
        before += b < (int)blockIdx.x ? c : 0;
      }
    at = block_exclusive(total, s_wave) + before;
  }
  rank_in_wave<ROUNDS>(key, live, a.shift, a.bits, cnt + wave * digits, off);
  __syncthreads();
  if (d < digits)
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w * digits + d];
      cnt[w * digits + d] = at;
      at += c;
    }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (64 * r + lane < live) {
      const int to = cnt[wave * digits + ((key[r] >> a.shift) & (digits - 1))] + off[r];
      a.key_out[to] = key[r];
      a.pos_out[to] = pos[r];
    }
}

// ------------------------------------------------------------------------------------------------------------- sums
struct SumArgs {
  const int* key; const int* pos; const void* dy; float* part; void* out;
  long V, lddy; int n, D, chunk, tpr_log2; float scale;
};

template <typename T, int VEC>
__device__ __forceinline__ void add_tokens(const SumArgs& a, int s, int e, int c, float (&acc)[VEC]) {
  const T* const dy = static_cast<const T*>(a.dy);
  for (int i = s; i < e; i += 8) {
    float v[8][VEC];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u < e) TkVec<T, VEC>::load(dy + a.pos[i + u] * a.lddy + c, v[u]);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u < e) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += v[u][k];
      }
  }
}

// Workgroup (chunk, column tile): the chunk's share of a row whose tokens cross the chunk's border; at most two do: the row
// of the chunk's first token (part 0) and, if it is another, the row of its last token (part 1).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_parts_kernel(SumArgs a) {
  const int lo = blockIdx.x * a.chunk, hi = min(a.n, lo + a.chunk), c = (blockIdx.y * 256 + threadIdx.x) * VEC;
  const int lane = threadIdx.x & 63;
  const int first = a.key[lo], last = a.key[hi - 1];
  int same_first = 0, same_last = 0;             // the keys are sorted: how many equal the first, the last
  for (int i = lo; i < hi; i += 64) {
    const int k = i + lane < hi ? a.key[i + lane] : -1;
    same_first += (int)__popcll(__ballot(k == first));
    same_last += (int)__popcll(__ballot(k == last));
  }
  if (c >= a.D) return;
  const bool left = lo > 0 && a.key[lo - 1] == first, right = hi < a.n && a.key[hi] == last;
  float* const part = a.part + (size_t)blockIdx.x * 2 * a.D + c;
  if (first < a.V && (left || (right && first == last))) {
    float acc[VEC] = {};
    add_tokens<T, VEC>(a, lo, lo + same_first, c, acc);
#pragma unroll
    for (int q = 0; q < VEC; ++q) part[q] = acc[q];
  }
  if (last < a.V && right && first != last) {
    float acc[VEC] = {};
    add_tokens<T, VEC>(a, hi - same_last, hi, c, acc);
#pragma unroll
    for (int q = 0; q < VEC; ++q) part[a.D + q] = acc[q];
  }
}

// Workgroup (32 table rows, column tile); 2^tpr_log2 threads a row.  The rows lie gridDim.x apart: frequent tokens often have
// neighbouring ids, and 32 frequent rows one after the other would be the launch's last workgroup (measured: 16384 tokens
// with frequencies 1 / k on 50001 x 1024, neighbouring rows 327 us).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_rows_kernel(SumArgs a) {
  __shared__ int s_key[257], s_at[2 * kRows];
  const int tid = threadIdx.x;
  // where each row's tokens start and end: a sample of 256 keys in LDS, then binary search between two of them
  const int per = (a.n + 255) / 256;
  s_key[tid] = per && (long)tid * per < a.n ? a.key[tid * per] : 0x7fffffff;
  __syncthreads();
  if (tid < 2 * kRows) {
    const long v = (long)blockIdx.x + (long)(tid >> 1) * gridDim.x + (tid & 1);
    int b = 0;                                   // samples below v
    for (int half = 128; half > 0; half >>= 1)
      if (s_key[b + half - 1] < v) b += half;
    if (b < 256 && s_key[b] < v) ++b;
    int lo = b > 0 ? (b - 1) * per : 0, len = b > 0 ? min(a.n - lo, per) : 0;
    while (len > 0) {
      const int half = len >> 1;
      if (a.key[lo + half] < v) { lo += half + 1; len -= half + 1; } else len = half;
    }
    s_at[tid] = lo;
  }
  __syncthreads();
  const int tpr = 1 << a.tpr_log2, t = tid & (tpr - 1);
  const int c = (blockIdx.y * tpr + t) * VEC;
  if (c >= a.D) return;
  T* const out = static_cast<T*>(a.out);
  for (int r = tid >> a.tpr_log2; r < kRows; r += 256 >> a.tpr_log2) {
    const long v = (long)blockIdx.x + (long)r * gridDim.x;
    if (v >= a.V) break;
    const int s = s_at[2 * r], e = s_at[2 * r + 1];
    float acc[VEC] = {};
    const int k0 = s / a.chunk, k1 = (e - 1) / a.chunk;
    if (e == s || k0 == k1) {
      add_tokens<T, VEC>(a, s, e, c, acc);
    } else {                                     // the row crosses a border: the chunks' parts, in order
      const float* const p = a.part + c;
      if (s > k0 * a.chunk) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] = p[((size_t)k0 * 2 + 1) * a.D + q];
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] = p[(size_t)k0 * 2 * a.D + q];
      }
      for (int k = k0 + 1; k <= k1; k += 8) {
        float v8[8][VEC];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int q = 0; q < VEC; ++q) v8[u][q] = k + u <= k1 ? p[(size_t)(k + u) * 2 * a.D + q] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int q = 0; q < VEC; ++q) acc[q] += v8[u][q];
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
  p.chunk = (int)std::min<int64_t>(std::max<int64_t>(32, n / 1024), 1024);
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
  SortArgs a = {ids, nullptr, nullptr, key_a, pos_a, reinterpret_cast<int*>(w + p.hist), (long)V, skip, (int)n, ids64, 0, p.bits, p.blocks, p.blocks > kScanBlocks};
  if (n > 0 && n <= kOne) {
    hipLaunchKernelGGL(emb_sort_one_kernel, dim3(1), dim3(kSortBlock), 0, s, a, p.passes);
  } else if (n > 0) {
    for (int k = 0; k < p.passes; ++k) {
      const bool to_a = ((p.passes - 1 - k) & 1) == 0;       // the last pass ends in a
      a.key_in = k == 0 ? nullptr : to_a ? key_b : key_a;
      a.pos_in = k == 0 ? nullptr : to_a ? pos_b : pos_a;
      a.key_out = to_a ? key_a : key_b;
      a.pos_out = to_a ? pos_a : pos_b;
      a.shift = k * p.bits;
      hipLaunchKernelGGL(emb_count_kernel, dim3(p.blocks), dim3(kSortBlock), 0, s, a);
      if (a.scanned) hipLaunchKernelGGL(emb_scan_kernel, dim3(1), dim3(kSortBlock), 0, s, a.hist, p.blocks << p.bits);
      hipLaunchKernelGGL(emb_scatter_kernel, dim3(p.blocks), dim3(kSortBlock), 0, s, a);
    }
  }
  const SumArgs q = {key_a, pos_a, dy, reinterpret_cast<float*>(w + p.part), out, (long)V, (long)lddy, (int)n, D, p.chunk, 0, scale};
  const int vec = dtype == TK_BF16 ? 8 : 4;
  const bool v = D % vec == 0 && lddy % vec == 0 && dtf_aligned16(dy) && dtf_aligned16(out);
  if (dtype == TK_BF16) v ? sums<unsigned short, 8>(q, p.chunks, s) : sums<unsigned short, 1>(q, p.chunks, s);
  else v ? sums<float, 4>(q, p.chunks, s) : sums<float, 1>(q, p.chunks, s);
  return dtf_check_launch();
}
