// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   forward    y[i] = scale table[id_i]                (an id outside the table gives a row of zeros)
//   backward   dtable[v] = scale sum_{i: id_i = v} dy[i]     for every row of the table, zeros where no token has it
//
// The gradient is a segmented sum.  Tokens are sorted by id, stably, so a row's tokens stand in the order of their
// positions; a row with tokens is then written by one workgroup: no atomics on floats (the same inputs give the same bits)
// and no fp32 table in between.
//   sort    LSD radix sort of (id, position) with digits of at most 9 bits (32 KB of counters): up to 8192 tokens in ONE
//           workgroup and launch, else count / scatter launches over blocks of 4096 tokens.  The sort keeps a few CUs busy;
//           the other workgroups of its launches fill the table's gradient with zeros meanwhile (measured apart: 39 us of
//           sorting 16384 tokens in one workgroup, 25 us of filling 50001 x 1024 bf16).
//   chunks  The sorted list is cut into chunks of 16 tokens or more, one workgroup (or part of one) each, so that frequent
//           rows are shared: rows inside a chunk are summed in fp32, scaled, rounded once and stored; of a row that crosses
//           the chunk's border (at most two do) the sum is kept as a part.
//   join    The chunk in which a crossing row starts adds the row's parts in order and stores it.
// Bound by memory: the table's gradient is written once (V D elements) and again where a row has tokens, dy is read once.
// 65536 tokens on 131072 x 1024 fp32: 106 us for the sort's launches with 512 MB of zeros beside it, 113 us for the chunks, 11 us
// for the join; small tables are bound by the launches' latency (16384 tokens on 50001 x 1024 bf16: 38, 12 and 6 us).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "token_ops.h"

namespace {
// tokens that one workgroup sorts: 8192 take 35 us that way (the whole gradient, 64 columns), 12288 take 44, and the launches
// over several workgroups 37
constexpr int kOne = 8192;
constexpr int kSortBlock = 1024, kSortWaves = kSortBlock / 64;
constexpr int kKeys = 4096;                      // tokens a workgroup of the multi-launch sort
constexpr int kMaxBits = 9;
constexpr int kScanBlocks = 256;                 // up to here a scatter block adds up the counts by itself

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

// Zeros for the 16-byte pieces [lo, hi) of the table's gradient, by the workgroups past the first `skip` of a launch.
struct Fill {
  tk_u32x4* out; long lo, hi;
};
__device__ __forceinline__ void fill_zero(const Fill& f, int skip) {
  const long step = (long)(gridDim.x - skip) * kSortBlock;
  for (long i = f.lo + (long)(blockIdx.x - skip) * kSortBlock + threadIdx.x; i < f.hi; i += step) f.out[i] = tk_u32x4{0u, 0u, 0u, 0u};
}

__global__ void emb_tail_kernel(char* out, int bytes) {
  if ((int)threadIdx.x < bytes) out[threadIdx.x] = 0;
}

struct SortArgs {
  const void* ids; const int* key_in; const int* pos_in; int* key_out; int* pos_out; int* hist;    // hist [digits][blocks]
  long V; long long skip; int n, ids64, shift, bits, blocks, scanned;
};

__device__ __forceinline__ int load_key(const SortArgs& a, int i) { return a.key_in ? a.key_in[i] : key_of(a.ids, a.ids64, i, a.V, a.skip); }

// Lanes of the wave whose digit equals this lane's (inactive lanes excluded): one ballot a bit.
__device__ __forceinline__ unsigned long long same_digit(int digit, int bits, bool active) {
  const unsigned long long act = __ballot(active);
  unsigned lo = (unsigned)act, hi = (unsigned)(act >> 32);
  for (int b = 0; b < bits; ++b) {
    const unsigned own = 0u - ((unsigned)(digit >> b) & 1u);          // all ones where this lane's bit is set
    const unsigned long long set = __ballot(own != 0u);
    lo &= ~((unsigned)set ^ own);
    hi &= ~((unsigned)(set >> 32) ^ own);
  }
  return ((unsigned long long)hi << 32) | lo;
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
    if (64 * r >= live) break;                   // the same for the whole wave
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
__global__ __launch_bounds__(kSortBlock) void emb_sort_one_kernel(SortArgs a, int passes, Fill f) {
  if (blockIdx.x > 0) return fill_zero(f, 1);
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

__global__ __launch_bounds__(kSortBlock) void emb_count_kernel(SortArgs a, Fill f) {
  if ((int)blockIdx.x >= a.blocks) return fill_zero(f, a.blocks);
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

__global__ __launch_bounds__(kSortBlock) void emb_scatter_kernel(SortArgs a, Fill f) {
  if ((int)blockIdx.x >= a.blocks) return fill_zero(f, a.blocks);
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
  long V, lddy; int n, D, chunk, chunks, tpr_log2; float scale;
};

// A chunk and a column tile belong to 2^tpr_log2 threads.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_chunks_kernel(SumArgs a) {
  const int tpr = 1 << a.tpr_log2, t = threadIdx.x & (tpr - 1);
  const int chunk = (int)((blockIdx.x * 256u + threadIdx.x) >> a.tpr_log2), c = (blockIdx.y * tpr + t) * VEC;
  if (chunk >= a.chunks || c >= a.D) return;
  const int lo = chunk * a.chunk, hi = min(a.n, lo + a.chunk);
  const T* const dy = static_cast<const T*>(a.dy) + c;
  T* const out = static_cast<T*>(a.out) + c;
  float* const part = a.part + (size_t)chunk * 2 * a.D + c;
  const int first = a.key[lo];
  bool inside = lo == 0 || a.key[lo - 1] != first;         // the current row starts in this chunk
  float acc[VEC] = {};
  int key[9], pos[8];
  auto fetch = [&](int i0) {                     // keys and positions of eight tokens, and the key behind them (-1: none)
#pragma unroll
    for (int u = 0; u < 9; ++u) key[u] = a.key[min(i0 + u, a.n - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) pos[u] = a.pos[min(i0 + u, a.n - 1)];
  };
  fetch(lo);
  for (int i0 = lo; i0 < hi; i0 += 8) {
    const int cnt = min(8, hi - i0);
    // every load is unconditional (tokens past the end repeat the last one), so that all eight rows are under way at once
    float v[8][VEC];
#pragma unroll
    for (int u = 0; u < 8; ++u) TkVec<T, VEC>::load(dy + pos[u] * a.lddy, v[u]);
    int now[9];
#pragma unroll
    for (int u = 0; u < 9; ++u) now[u] = i0 + u < a.n ? key[u] : -1;
    fetch(i0 + 8);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (u >= cnt || now[u] >= a.V) continue;   // tokens without a gradient are sorted behind all others
#pragma unroll
      for (int q = 0; q < VEC; ++q) acc[q] += v[u][q];
      const bool ends = now[u + 1] != now[u];
      if (!ends && i0 + u + 1 < hi) continue;
      if (ends && inside) {
        float o[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) o[q] = acc[q] * a.scale;
        TkVec<T, VEC>::store(out + (long)now[u] * a.D, o);
      } else {                                   // part 0: of the chunk's first row, part 1: of its last, if it is another
        float* const p = part + (now[u] == first ? 0 : a.D);
#pragma unroll
        for (int q = 0; q < VEC; ++q) p[q] = acc[q];
      }
#pragma unroll
      for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
      inside = true;
    }
  }
}

// Workgroup (chunk, 64 pieces of columns); the four waves take a quarter of the row's parts each, in order.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_join_kernel(SumArgs a) {
  __shared__ float s_acc[3][64][VEC];
  const int chunk = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (blockIdx.y * 64 + lane) * VEC;
  const int lo = chunk * a.chunk, hi = min(a.n, lo + a.chunk);
  const int v = a.key[hi - 1];
  if (v >= a.V || hi == a.n || a.key[hi] != v) return;                 // the last row ends here
  const bool whole = a.key[lo] == v;
  if (whole && lo > 0 && a.key[lo - 1] == v) return;                   // it started before this chunk
  int last = chunk;                              // the last chunk that begins with this row
  while (true) {
    const int k = last + 1 + lane;
    const unsigned long long m = __ballot(k < a.chunks && a.key[min(k, a.chunks - 1) * a.chunk] == v);
    last += m == ~0ull ? 64 : (int)__builtin_ctzll(~m);
    if (m != ~0ull) break;
  }
  const float* const p = a.part + (c < a.D ? c : 0);
  const int count = last - chunk + 1, per = (count + 3) >> 2, k0 = chunk + wave * per, k1 = min(last + 1, k0 + per);
  float acc[VEC] = {};
  for (int k = k0; k < k1; k += 8) {
    float v8[8][VEC];
#pragma unroll
    for (int u = 0; u < 8; ++u) {                // past the end: the last part again, not added
      const int at = min(k + u, last);
      const float* const q8 = p + ((size_t)at * 2 + (at == chunk && !whole ? 1 : 0)) * a.D;
#pragma unroll
      for (int q = 0; q < VEC; ++q) v8[u][q] = q8[q];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int q = 0; q < VEC; ++q) acc[q] += k + u < k1 ? v8[u][q] : 0.f;
  }
  if (wave) {
#pragma unroll
    for (int q = 0; q < VEC; ++q) s_acc[wave - 1][lane][q] = acc[q];
  }
  __syncthreads();                               // every wave took the same way here
  if (wave || c >= a.D) return;
#pragma unroll
  for (int q = 0; q < VEC; ++q) acc[q] = (((acc[q] + s_acc[0][lane][q]) + s_acc[1][lane][q]) + s_acc[2][lane][q]) * a.scale;
  TkVec<T, VEC>::store(static_cast<T*>(a.out) + (long)v * a.D + c, acc);
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
  p.chunk = (int)std::min<int64_t>(std::max<int64_t>(16, n / 2048), 1024);
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
  if (n < 0 || n > (1ll << 25) || V <= 0 || V > (1ll << 30) || D <= 0 || D > (1 << 20)) return DTF_ERR_SHAPE;
  return DTF_OK;
}

int row_threads_log2(int D, int vec, int most) {
  int l = 0;
  while ((1 << l) * vec < D && (1 << l) < most) ++l;
  return l;
}

template <typename T, int VEC>
void sums(const SumArgs& in, hipStream_t s) {
  SumArgs a = in;
  a.tpr_log2 = row_threads_log2(a.D, VEC, 256);
  hipLaunchKernelGGL((emb_chunks_kernel<T, VEC>), dim3((unsigned)((((long)a.chunks << a.tpr_log2) + 255) / 256), dtf_cdiv(a.D, VEC << a.tpr_log2)), dim3(256), 0, s, a);
  if (a.chunks > 1) hipLaunchKernelGGL((emb_join_kernel<T, VEC>), dim3(a.chunks - 1, dtf_cdiv(a.D, 64 * VEC)), dim3(256), 0, s, a);
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
  if (!dtf_aligned16(out)) return DTF_ERR_ALIGN;
  const EmbPlan p = plan(n, V, D);
  if (n > 0 && ws_bytes < (int64_t)p.total) return DTF_ERR_SHAPE;
  char* const w = static_cast<char*>(ws);
  int* const key_a = reinterpret_cast<int*>(w + p.key_a), * const pos_a = reinterpret_cast<int*>(w + p.pos_a);
  int* const key_b = reinterpret_cast<int*>(w + p.key_b), * const pos_b = reinterpret_cast<int*>(w + p.pos_b);
  SortArgs a = {ids, nullptr, nullptr, key_a, pos_a, reinterpret_cast<int*>(w + p.hist), (long)V, skip, (int)n, ids64, 0, p.bits, p.blocks, p.blocks > kScanBlocks};
  // zeros, in equal shares of the sort's launches; the bytes behind the last whole 16-byte piece by themselves
  const int64_t bytes = V * D * (dtype == TK_BF16 ? 2 : 4), pieces = bytes / 16;
  const int shares = n <= kOne ? 1 : 2 * p.passes;
  auto fill = [&](int share) { return Fill{static_cast<tk_u32x4*>(out), (long)(pieces * share / shares), (long)(pieces * (share + 1) / shares)}; };
  const int64_t most = (pieces + shares - 1) / shares;        // pieces of the largest share
  const unsigned fillers = (unsigned)std::min<int64_t>(511, (most + kSortBlock - 1) / kSortBlock);
  if (bytes % 16) hipLaunchKernelGGL(emb_tail_kernel, dim3(1), dim3(64), 0, s, static_cast<char*>(out) + pieces * 16, (int)(bytes % 16));
  if (n <= kOne) {
    hipLaunchKernelGGL(emb_sort_one_kernel, dim3(1 + fillers), dim3(kSortBlock), 0, s, a, n > 0 ? p.passes : 0, fill(0));
  } else {
    for (int k = 0; k < p.passes; ++k) {
      const bool to_a = ((p.passes - 1 - k) & 1) == 0;       // the last pass ends in a
      a.key_in = k == 0 ? nullptr : to_a ? key_b : key_a;
      a.pos_in = k == 0 ? nullptr : to_a ? pos_b : pos_a;
      a.key_out = to_a ? key_a : key_b;
      a.pos_out = to_a ? pos_a : pos_b;
      a.shift = k * p.bits;
      hipLaunchKernelGGL(emb_count_kernel, dim3(p.blocks + fillers), dim3(kSortBlock), 0, s, a, fill(2 * k));
      if (a.scanned) hipLaunchKernelGGL(emb_scan_kernel, dim3(1), dim3(kSortBlock), 0, s, a.hist, p.blocks << p.bits);
      hipLaunchKernelGGL(emb_scatter_kernel, dim3(p.blocks + fillers), dim3(kSortBlock), 0, s, a, fill(2 * k + 1));
    }
  }
  if (n > 0) {
    const SumArgs q = {key_a, pos_a, dy, reinterpret_cast<float*>(w + p.part), out, (long)V, (long)lddy, (int)n, D, p.chunk, p.chunks, 0, scale};
    const int vec = dtype == TK_BF16 ? 8 : 4;
    const bool v = D % vec == 0 && lddy % vec == 0 && dtf_aligned16(dy);
    if (dtype == TK_BF16) v ? sums<unsigned short, 8>(q, s) : sums<unsigned short, 1>(q, s);
    else v ? sums<float, 4>(q, s) : sums<float, 1>(q, s);
  }
  return dtf_check_launch();
}
