// Row lookup with scaling and its gradient by sorted ids (nof_embed_fwd / nof_embed_bwd, include/nof_hip.h).
//
//   out[i, :]  = scale * table[ids[i], :]                    an id outside [0, V): a row of zeros
//   grad[v, :] = scale * sum over {i : ids[i] = v} dout[i, :]  an id outside [0, V): no contribution; a row nobody names: zeros
//
// Both are bound by memory: the rows read and written once each.  The gradient adds in a fixed order, so equal inputs give equal
// bits (the hash table's scatter beside it, nof_hash.hip, adds with atomics):
//   1. a stable radix sort of (id, position): one k_embed_hist + k_embed_scatter per digit, or k_embed_sort_small as one workgroup;
//   2. k_embed_reduce: a group of lanes owns a run of C sorted positions and one slice of the columns, reads the rows of dout behind
//      them and writes the sum of every id that lies within the run; an id cut by the run's ends leaves a partial sum.  Further
//      workgroups of the same launch write the zeros of the rows that no id names -- most of the bytes of a large table -- where the
//      sort's launches have not done so;
//   3. k_embed_join: the partial sums of a cut id, in the order of their runs.
// Few positions of few rows take one launch instead (k_embed_few).
#include "nof_learn_dev.h"

#define EMB_T 256                       // threads of the streaming kernels
#define EMB_ZROWS 32                    // table rows per workgroup of the zero role at a time
#define EMB_ZBYTES 65536                // of the sort's zero role per workgroup
#define EMB_ZHIST ((int64_t)12 << 20)     // bytes of zeros that ride in one launch of the sort
#define EMB_ZSCATTER ((int64_t)32 << 20)
#define EMB_ZSMALL ((int64_t)48 << 20)
#define EMB_SMALL 4096                  // positions that the one-workgroup sort holds in LDS
#define EMB_SORT_T 512
#define EMB_SORT_W (EMB_SORT_T / 64)
#define EMB_BITS 10                     // widest digit of the many-workgroup sort
#define EMB_MAX_BLOCKS 128
#define EMB_MAX_GRID (1 << 22)          // workgroups of a role whose work has no such limit: a launch has less than 2^32 threads on an axis
#define EMB_FEW_N 4096                  // positions that k_embed_few lists

// ---- lookup -----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t emb_id(const void* __restrict__ ids, int ids64, int64_t i) {
  return ids64 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

// 16 bytes of a row per access, wherever the row starts: gfx950 takes them at any border, and rows of odd length would otherwise go one
// element at a time.  The last access of a row may be short (n < V elements, the others as zeros).
template <typename T> struct EmbVec { static constexpr int V = 16 / (int)sizeof(T); };
typedef uint32_t emb_u4 __attribute__((ext_vector_type(4)));
template <int SIZE> struct EmbAt;
template <> struct EmbAt<2> { typedef emb_u4 t __attribute__((aligned(2))); };
template <> struct EmbAt<4> { typedef emb_u4 t __attribute__((aligned(4))); };
template <typename T> using EmbBits = typename EmbAt<sizeof(T)>::t;
// ONCE: past the caches, for what is read only here and is too large to lie in them from its making (the gradient's rows: emb_launch_sums)
template <typename T, int V, bool ONCE>
__device__ __forceinline__ void emb_load(const T* __restrict__ p, int n, float (&f)[V]) {
  if (n >= V) {
    const EmbBits<T>* at = reinterpret_cast<const EmbBits<T>*>(p);
    const emb_u4 bits = ONCE ? __builtin_nontemporal_load(at) : *at;
    const LearnVec<T, V> x = __builtin_bit_cast(LearnVec<T, V>, bits);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = lf(x.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < n ? lf(p[i]) : 0.0f;
  }
}
// a store past the caches: nothing here reads it again, and the rows that are read stay (65536 x 2048 bf16 looked up: 59 us, 91 without;
// the gradient of a 131072-row table by them: 26 us less)
template <typename T, int V>
__device__ __forceinline__ void emb_store(T* __restrict__ p, int n, const float (&f)[V]) {
  if (n >= V) {
    LearnVec<T, V> x;
#pragma unroll
    for (int i = 0; i < V; ++i) x.v[i] = lt<T>(f[i]);
    __builtin_nontemporal_store(__builtin_bit_cast(emb_u4, x), reinterpret_cast<EmbBits<T>*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = lt<T>(f[i]);
  }
}

// 2^ls lanes a row, further columns by blockIdx.y
template <typename T>
__global__ __launch_bounds__(EMB_T) void k_embed_fwd(const T* __restrict__ table, int64_t stride, const void* __restrict__ ids, int ids64,
                                                     float scale, T* __restrict__ out, int64_t N, int64_t rows, int D, int ls) {
  constexpr int V = EmbVec<T>::V;
  const int lane = threadIdx.x & ((1 << ls) - 1);
  const int col = (((int)blockIdx.y << ls) + lane) * V;
  const int64_t step = (int64_t)gridDim.x * (EMB_T >> ls);
  if (col >= D) return;
  for (int64_t i = (int64_t)blockIdx.x * (EMB_T >> ls) + (threadIdx.x >> ls); i < N; i += step) {
    const int64_t id = emb_id(ids, ids64, i);
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = 0.0f;
    if (id >= 0 && id < rows) {
      emb_load<T, V, false>(table + id * stride + col, D - col, f);
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] *= scale;
    }
    emb_store<T, V>(out + i * D + col, D - col, f);
  }
}

// ---- stable radix sort of (id, position) ------------------------------------------------------------------------------------------
// An absent id sorts behind every row as the key V.
__device__ __forceinline__ uint32_t emb_key(const void* __restrict__ ids, int ids64, int64_t i, int64_t rows) {
  const int64_t id = emb_id(ids, ids64, i);
  return id >= 0 && id < rows ? (uint32_t)id : (uint32_t)rows;
}

// the lanes of this wave that are `in` and hold the same digit as this lane
__device__ __forceinline__ uint64_t emb_match(uint32_t digit, int bits, bool in) {
  uint64_t m = __ballot(in);
  for (int b = 0; b < bits; ++b) {
    const bool one = (digit >> b) & 1u;
    const uint64_t bal = __ballot(in && one);
    m &= one ? bal : ~bal;
  }
  return m;
}

// Zeros for the gradient's first rows, written by workgroups that ride behind the sort's own: those few leave the chip idle for as long as
// the memory takes for tens of megabytes (named rows are overwritten later).  131072 x 2048 bf16 196 us without, 190 so; 200000 x 64 fp32 by
// 2000 positions 32 and 25, a million by 100000 x 64 bf16 159 and 146.
struct EmbZero { char* at; uint64_t bytes; };                         // any border, whole elements
__device__ __forceinline__ void emb_zero(const EmbZero& z, uint32_t block, uint32_t threads) {
  const uint64_t lo = (uint64_t)block * EMB_ZBYTES, hi = lo + EMB_ZBYTES < z.bytes ? lo + EMB_ZBYTES : z.bytes, whole = lo + (hi - lo) / 16 * 16;
  const emb_u4 none = {0, 0, 0, 0};
  for (uint64_t i = lo + threadIdx.x * 16; i < whole; i += (uint64_t)threads * 16) __builtin_nontemporal_store(none, reinterpret_cast<EmbAt<2>::t*>(z.at + i));
  for (uint64_t i = whole + threadIdx.x * 2; i < hi; i += (uint64_t)threads * 2) *reinterpret_cast<uint16_t*>(z.at + i) = 0;
}

struct EmbSort {
  const void* ids; int ids64; int64_t rows;
  uint32_t N, per;                      // positions; positions per workgroup (a multiple of EMB_SORT_T)
  int n_blocks, passes, bits;
};

// hist[block][digit] of a pass.  (Counted with atomics by the scatter before instead, an id that many positions hold is one address:
// 15 us for 8192 positions against 8 + 3.)
__global__ __launch_bounds__(EMB_SORT_T) void k_embed_hist(EmbSort s, int pass, const uint32_t* __restrict__ key_in, uint32_t* __restrict__ hist, EmbZero z) {
  if ((int)blockIdx.x >= s.n_blocks) return emb_zero(z, blockIdx.x - s.n_blocks, EMB_SORT_T);
  __shared__ uint32_t cnt[1 << EMB_BITS];
  const int bins = 1 << s.bits, shift = pass * s.bits;
  for (int d = threadIdx.x; d < bins; d += EMB_SORT_T) cnt[d] = 0;
  __syncthreads();
  const uint32_t lo = blockIdx.x * s.per, hi = lo + s.per < s.N ? lo + s.per : s.N;
  for (uint32_t i = lo + threadIdx.x; i < hi; i += EMB_SORT_T) {
    const uint32_t k = pass == 0 ? emb_key(s.ids, s.ids64, i, s.rows) : key_in[i];
    atomicAdd(&cnt[(k >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += EMB_SORT_T) hist[blockIdx.x * bins + d] = cnt[d];
}

// One digit: a workgroup knows where its keys go from the histogram of all workgroups (at most EMB_MAX_BLOCKS * 4 KiB, from L2), a
// wave from the counts of the waves before it, a lane from its rank among the equal digits of its wave: no order is left to chance.
__global__ __launch_bounds__(EMB_SORT_T) void k_embed_scatter(EmbSort s, int pass, const uint32_t* __restrict__ key_in,
                                                              const uint32_t* __restrict__ pos_in, uint32_t* __restrict__ key_out,
                                                              uint32_t* __restrict__ pos_out, const uint32_t* __restrict__ hist, EmbZero z) {
  if ((int)blockIdx.x >= s.n_blocks) return emb_zero(z, blockIdx.x - s.n_blocks, EMB_SORT_T);
  __shared__ uint32_t cnt[EMB_SORT_W][1 << EMB_BITS];
  __shared__ uint32_t wsum[EMB_SORT_W];
  const int bins = 1 << s.bits, shift = pass * s.bits, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t lo = blockIdx.x * s.per, hi = lo + s.per < s.N ? lo + s.per : s.N, per_wave = s.per / EMB_SORT_W;
  const uint32_t wlo = lo + w * per_wave < hi ? lo + w * per_wave : hi, whi = wlo + per_wave < hi ? wlo + per_wave : hi;
  for (int d = threadIdx.x; d < bins * EMB_SORT_W; d += EMB_SORT_T) cnt[d >> s.bits][d & (bins - 1)] = 0;
  __syncthreads();
  for (uint32_t i = wlo + lane; i < whi; i += 64) {
    const uint32_t k = pass == 0 ? emb_key(s.ids, s.ids64, i, s.rows) : key_in[i];
    atomicAdd(&cnt[w][(k >> shift) & (bins - 1)], 1u);
  }
  // digits 2t and 2t + 1 are thread t's (bins <= 2 * EMB_SORT_T): totals over all workgroups, and over those before this one
  uint32_t tot[2] = {0, 0}, before[2] = {0, 0};
  const int d0 = 2 * threadIdx.x;
  if (d0 < bins) {
#pragma unroll 16                        // (sixteen loads in flight: one at a time is a trip to L2 per workgroup of the sort)
    for (int b = 0; b < s.n_blocks; ++b) {
      const uint2 x = *reinterpret_cast<const uint2*>(hist + (size_t)b * bins + d0);
      tot[0] += x.x; tot[1] += x.y;
      if (b < (int)blockIdx.x) { before[0] += x.x; before[1] += x.y; }
    }
  }
  uint32_t run = tot[0] + tot[1];
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(run, o);
    if (lane >= o) run += y;
  }
  if (lane == 63) wsum[w] = run;
  __syncthreads();
  uint32_t at = run - tot[0] - tot[1];
  for (int k = 0; k < w; ++k) at += wsum[k];
  if (d0 < bins) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t next = at + before[q];
      for (int k = 0; k < EMB_SORT_W; ++k) {
        const uint32_t c = cnt[k][d0 + q];
        cnt[k][d0 + q] = next;
        next += c;
      }
      at += tot[q];
    }
  }
  __syncthreads();
  for (uint32_t base = wlo; base < whi; base += 64) {
    const uint32_t i = base + lane;
    const bool in = i < whi;
    uint32_t k = 0, p = 0;
    if (in) {
      k = pass == 0 ? emb_key(s.ids, s.ids64, i, s.rows) : key_in[i];
      p = pass == 0 ? i : pos_in[i];
    }
    const uint32_t digit = (k >> shift) & (bins - 1);
    const uint64_t same = emb_match(digit, s.bits, in);
    const int leader = in ? __ffsll((unsigned long long)same) - 1 : lane;
    uint32_t old = 0;
    if (in && lane == leader) old = atomicAdd(&cnt[w][digit], (uint32_t)__popcll(same));
    old = __shfl(old, leader);
    if (in) {
      const uint32_t to = old + (uint32_t)__popcll(same & (((uint64_t)1 << lane) - 1));
      key_out[to] = k;
      pos_out[to] = p;
    }
  }
}

// The whole sort as one workgroup of sixteen waves, 8 bits a digit, keys and positions in LDS (56 KiB).
__global__ __launch_bounds__(1024) void k_embed_sort_small(const void* __restrict__ ids, int ids64, int64_t rows, int N, int passes,
                                                           uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out, EmbZero z) {
  if (blockIdx.x > 0) return emb_zero(z, blockIdx.x - 1, 1024);
  __shared__ uint32_t key[2][EMB_SMALL];
  __shared__ uint16_t pos[2][EMB_SMALL];
  __shared__ uint32_t cnt[16][128];                                  // two digits a word: counts stay below 2^16
  __shared__ uint32_t wsum[2];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int per_wave = ((N + 1023) / 1024) * 64, wlo = w * per_wave < N ? w * per_wave : N, whi = wlo + per_wave < N ? wlo + per_wave : N;
  for (int i = threadIdx.x; i < N; i += 1024) { key[0][i] = emb_key(ids, ids64, i, rows); pos[0][i] = (uint16_t)i; }
  int cur = 0;
  for (int pass = 0; pass < passes; ++pass, cur ^= 1) {
    for (int d = threadIdx.x; d < 16 * 128; d += 1024) cnt[d >> 7][d & 127] = 0;
    __syncthreads();
    for (int i = wlo + lane; i < whi; i += 64) {
      const uint32_t g = (key[cur][i] >> (8 * pass)) & 255u;
      atomicAdd(&cnt[w][g >> 1], 1u << (16 * (g & 1)));
    }
    __syncthreads();
    // thread t < 128 owns digits 2t and 2t + 1
    uint32_t tot = 0, tot2 = 0, run = 0;
    const int d = threadIdx.x;
    if (d < 128) {
      for (int k = 0; k < 16; ++k) { tot += cnt[k][d] & 0xffffu; tot2 += cnt[k][d] >> 16; }
      run = tot + tot2;
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(run, o);
        if (lane >= o) run += y;
      }
      if (lane == 63) wsum[w] = run;
    }
    __syncthreads();
    if (d < 128) {
      uint32_t next = run - tot - tot2 + (w == 1 ? wsum[0] : 0u), next2 = next + tot;
      for (int k = 0; k < 16; ++k) {
        const uint32_t c = cnt[k][d];
        cnt[k][d] = next | (next2 << 16);
        next += c & 0xffffu;
        next2 += c >> 16;
      }
    }
    __syncthreads();
    for (int base = wlo; base < whi; base += 64) {
      const int i = base + lane;
      const bool in = i < whi;
      const uint32_t k = in ? key[cur][i] : 0u, g = (k >> (8 * pass)) & 255u;
      const uint64_t same = emb_match(g, 8, in);
      const int leader = in ? __ffsll((unsigned long long)same) - 1 : lane;
      uint32_t old = 0;
      if (in && lane == leader) old = atomicAdd(&cnt[w][g >> 1], (uint32_t)__popcll(same) << (16 * (g & 1)));
      old = (__shfl(old, leader) >> (16 * (g & 1))) & 0xffffu;
      if (in) {
        const int to = (int)old + __popcll(same & (((uint64_t)1 << lane) - 1));
        key[cur ^ 1][to] = k;
        pos[cur ^ 1][to] = pos[cur][i];
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < N; i += 1024) { key_out[i] = key[cur][i]; pos_out[i] = pos[cur][i]; }
}

// ---- sums over the sorted positions -----------------------------------------------------------------------------------------------
// first position whose key is >= v
__device__ __forceinline__ uint32_t emb_lower(const uint32_t* __restrict__ key, uint32_t n, uint32_t v) {
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + ((hi - lo) >> 1);
    if (key[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

template <typename T, int V>
__device__ __forceinline__ void emb_put(T* __restrict__ grad, int64_t row, int D, int col, float scale, const float (&acc)[V]) {
  float f[V];
#pragma unroll
  for (int k = 0; k < V; ++k) f[k] = acc[k] * scale;
  emb_store<T, V>(grad + row * D + col, D - col, f);
}

// part [chunk][2][DP], DP = D up to a multiple of 8: the sum of the id that a run inherits from the run before it, and of the one that it starts and hands on
template <typename T, bool ONCE>
__global__ __launch_bounds__(EMB_T) void k_embed_reduce(const T* __restrict__ dout, int64_t stride, const uint32_t* __restrict__ key,
                                                        const uint32_t* __restrict__ pos, uint32_t N, uint32_t rows, int D, float scale,
                                                        T* __restrict__ grad, float* __restrict__ part, int ls, int C, uint32_t n_red, uint32_t zeroed) {
  constexpr int V = EmbVec<T>::V;
  const int DP = (D + 7) & ~7;
  const int lane = threadIdx.x & ((1 << ls) - 1);
  const int col = (((int)blockIdx.y << ls) + lane) * V;
  if (blockIdx.x >= n_red) {                                          // the zero role
    __shared__ uint8_t named[EMB_ZROWS];
    float z[V];
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = 0.0f;
    for (uint32_t v0 = zeroed + (blockIdx.x - n_red) * EMB_ZROWS; v0 < rows; v0 += (gridDim.x - n_red) * EMB_ZROWS) {        // (rows < 2^30: no overflow)
      if (threadIdx.x < EMB_ZROWS) {
        const uint32_t v = v0 + threadIdx.x;
        const uint32_t at = v < rows ? emb_lower(key, N, v) : 0;
        named[threadIdx.x] = v >= rows || (at < N && key[at] == v);
      }
      __syncthreads();
      if (col < D)
        for (int r = threadIdx.x >> ls; r < EMB_ZROWS; r += EMB_T >> ls)
          if (!named[r]) emb_store<T, V>(grad + (int64_t)(v0 + r) * D + col, D - col, z);
      __syncthreads();
    }
    return;
  }
  const uint32_t chunk = blockIdx.x * (EMB_T >> ls) + (threadIdx.x >> ls);
  const uint64_t first = (uint64_t)chunk * C;
  if (first >= N || col >= D) return;
  const uint32_t lo = (uint32_t)first, hi = N - lo > (uint32_t)C ? lo + C : N;
  uint32_t cur = key[lo];
  if (cur >= rows) return;                                            // absent ids are last
  bool inherited = lo > 0 && key[lo - 1] == cur;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;
  constexpr int U = 8;                                                // rows in flight per group
  uint32_t next_key[U], next_pos[U];                                  // (keys and positions a turn ahead: rows wait for one load, not for three)
  auto ahead = [&](uint32_t i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      next_key[u] = i + u < hi ? key[i + u] : rows;
      next_pos[u] = i + u < hi ? pos[i + u] : 0;
    }
  };
  ahead(lo);
  for (uint32_t i = lo; i < hi; i += U) {
    uint32_t kk[U];
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      kk[u] = next_key[u];
      if (kk[u] < rows) emb_load<T, V, ONCE>(dout + (int64_t)next_pos[u] * stride + col, D - col, x[u]);
    }
    ahead(i + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kk[u] != cur) {                                             // an id ends here (or the run does: `rows`)
        if (cur < rows && i + u < hi) {
          if (inherited) lstore<float, V>(part + ((size_t)chunk * 2) * DP + col, acc);
          else emb_put<T, V>(grad, cur, D, col, scale, acc);
          inherited = false;
          cur = kk[u];
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] = 0.0f;
        }
      }
      if (kk[u] < rows) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += x[u][k];
      }
    }
  }
  if (cur >= rows) return;
  const bool on = hi < N && key[hi] == cur;
  if (inherited) lstore<float, V>(part + ((size_t)chunk * 2) * DP + col, acc);
  else if (on) lstore<float, V>(part + ((size_t)chunk * 2 + 1) * DP + col, acc);
  else emb_put<T, V>(grad, cur, D, col, scale, acc);
}

// The run in which a cut id starts adds what the runs behind it inherited: a workgroup per run and slice of at most 64 x V columns, whose
// groups of lanes each add a stretch of the runs; their sums meet in LDS, neighbours first.  (One group for all of an id that many runs hold
// is a chain of loads: 17 us for the large table, 8 so.)
template <typename T>
__global__ __launch_bounds__(EMB_T) void k_embed_join(const uint32_t* __restrict__ key, uint32_t N, uint32_t rows, int D, float scale,
                                                      T* __restrict__ grad, const float* __restrict__ part, int ls, int C) {
  constexpr int V = 4;
  const int DP = (D + 7) & ~7;
  __shared__ float sums[EMB_T * V];
  const int lane = threadIdx.x & ((1 << ls) - 1), group = threadIdx.x >> ls, groups = EMB_T >> ls;
  const int col = (((int)blockIdx.y << ls) + lane) * V;
  for (uint32_t chunk = blockIdx.x;; chunk += gridDim.x) {              // (at most 2^28 runs: no overflow)
    const uint64_t first = (uint64_t)chunk * C, end = first + C;
    if (end >= N) return;
    const uint32_t lo = (uint32_t)first, id = key[end - 1], after = key[end], start = key[lo], before = key[lo > 0 ? lo - 1 : 0];
    if (id >= rows || after != id) continue;                            // nothing handed on
    if (start == id && lo > 0 && before == id) continue;                // nor started here
    uint32_t last = chunk;                                              // the last run that starts with the id, as many runs at a time as threads
    for (int more = EMB_T; more == EMB_T; last += more) {
      const uint64_t at = ((uint64_t)last + 1 + threadIdx.x) * C;
      more = __syncthreads_count(at < N && key[at] == id);
    }
    const uint32_t each = (last - chunk + groups - 1) / groups, c0 = chunk + 1 + group * each, c1 = c0 + each <= last ? c0 + each : last + 1;
    float acc[V], x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    if (col < D) {
      if (group == 0) lload<float, V>(part + ((size_t)chunk * 2 + 1) * DP + col, acc);
#pragma unroll 4
      for (uint32_t c = c0; c < c1; ++c) {
        lload<float, V>(part + ((size_t)c * 2) * DP + col, x);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += x[k];
      }
    }
    for (int o = 1; o < groups && o <= (int)(last - chunk - 1); o *= 2) {
#pragma unroll
      for (int k = 0; k < V; ++k) sums[threadIdx.x * V + k] = acc[k];
      __syncthreads();
      if ((group & (2 * o - 1)) == 0 && group + o < groups) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += sums[(threadIdx.x + (o << ls)) * V + k];
      }
      __syncthreads();
    }
    if (group == 0 && col < D) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (col + k < D) grad[(int64_t)id * D + col + k] = lt<T>(acc[k] * scale);
    }
  }
}

// ---- few rows, few positions ------------------------------------------------------------------------------------------------------
// One launch, no sort: a workgroup per table row and slice of the columns looks all ids over -- its waves a stretch each, keeping the
// positions that name the row in their order --, then its groups of lanes add a stretch of them each and their sums meet in LDS.  64 rows,
// 4096 positions of 16 fp32: 9 us, where the sort, its sums and their join take 18.
template <typename T>
__global__ __launch_bounds__(EMB_T) void k_embed_few(const T* __restrict__ dout, int64_t stride, const void* __restrict__ ids, int ids64, int N, int D,
                                                     float scale, T* __restrict__ grad, int ls) {
  constexpr int V = EmbVec<T>::V, W = EMB_T / 64;
  __shared__ uint16_t list[EMB_FEW_N + 64 * W];
  __shared__ int counts[W];
  __shared__ float sums[EMB_T * V];
  const int row = blockIdx.x, w = threadIdx.x >> 6, l64 = threadIdx.x & 63;
  const int per_wave = (N + EMB_T - 1) / EMB_T * 64, lo = w * per_wave, hi = lo + per_wave < N ? lo + per_wave : N;
  int count = 0;
#pragma unroll 8
  for (int base = lo; base < hi; base += 64) {
    const int i = base + l64;
    const bool mine = i < hi && emb_id(ids, ids64, i) == row;
    const uint64_t all = __ballot(mine);
    if (mine) list[lo + count + __popcll(all & (((uint64_t)1 << l64) - 1))] = (uint16_t)i;
    count += __popcll(all);
  }
  if (l64 == 0) counts[w] = count;
  __syncthreads();
  int total = 0, ends[W];
#pragma unroll
  for (int k = 0; k < W; ++k) { total += counts[k]; ends[k] = total; }
  const int lane = threadIdx.x & ((1 << ls) - 1), group = threadIdx.x >> ls, groups = EMB_T >> ls;
  const int col = (((int)blockIdx.y << ls) + lane) * V;
  const int each = (total + groups - 1) / groups, m0 = group * each, m1 = m0 + each < total ? m0 + each : total;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;
  if (col < D) {
    constexpr int U = 8;                                              // rows in flight per group
    for (int m = m0; m < m1; m += U) {
      float x[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = m + u < m1 ? m + u : m1 - 1;
        int at = q;                                                   // of the concatenated lists
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
          if (q >= ends[k]) at = q - ends[k] + (k + 1) * per_wave;
        emb_load<T, V, false>(dout + (int64_t)list[at] * stride + col, D - col, x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += m + u < m1 ? x[u][k] : 0.0f;
    }
  }
  for (int o = 1; o < groups && o <= total; o *= 2) {                 // (groups behind the last position hold zeros)
#pragma unroll
    for (int k = 0; k < V; ++k) sums[threadIdx.x * V + k] = acc[k];
    __syncthreads();
    if ((group & (2 * o - 1)) == 0 && group + o < groups) {
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += sums[(threadIdx.x + (o << ls)) * V + k];
    }
    __syncthreads();
  }
  if (group == 0 && col < D) emb_put<T, V>(grad, row, D, col, scale, acc);
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
// Sorted positions per run: as many as leave 2048 waves (two per SIMD).  A shorter run is more partial sums, a longer one a longer chain of
// loads.  Gradient alone, 8 / 16 / 32 / 64 positions: 8192 x 1024 bf16 40.7 / 41.5 / 46.6 / 57.8 us, 65536 x 256 fp32 57 / 43 / 37.7 / 39.1,
// 65536 x 2048 bf16 234 / 214 / 197 / 190.
static int emb_chunk(int64_t N, int32_t D, int size) {
  const int64_t nv = nof_div_up(D, 16 / size), waves = (N << learn_log2_up(nv < EMB_T ? nv : EMB_T)) * nof_div_up(nv, EMB_T) / 64;
  int c = 8;
  while (c < 64 && waves / (2 * c) >= 2048) c *= 2;
  return c;
}

struct EmbPlan {
  EmbSort s;
  bool few, small;
  int64_t key[2], pos[2], hist, part, bytes, zeroed;                  // zeroed: rows that the sort's launches clear
  int C, ls;                                                          // positions a run; 2^ls lanes a row
  uint32_t chunks, n_red;                                             // runs; workgroups that add them
};

// k_embed_few: every row's workgroups look all ids over, so few positions and rows x slices.  Against the sort: 4096 positions, 64 rows of 16
// fp32 9 us and 18 (15 and 21 if all name one row), 4096 rows of 32 16 and 24, 8000 of 16 25 and 24; 256 positions, 16000 rows 13 and 16;
// 8192 positions of 64 fp32 in 2 rows 32 and 22.
static bool emb_few(int64_t N, int64_t rows, int32_t D) { return N <= EMB_FEW_N && rows * nof_div_up(D, 32) * (N + 1024) <= (int64_t)20 << 20; }

static EmbPlan emb_plan(int64_t N, int64_t rows, int32_t D, int size) {
  EmbPlan p = {};
  const int bits = learn_log2_up(rows + 1) > 0 ? learn_log2_up(rows + 1) : 1;
  p.s.N = (uint32_t)N;
  p.s.rows = rows;
  p.few = emb_few(N, rows, D);
  if (p.few) {
    p.bytes = N > 0 ? 256 : 0;                                        // unused; a caller passes a workspace whatever the sizes
    return p;
  }
  p.small = N <= EMB_SMALL;
  if (p.small) {
    p.s.passes = (bits + 7) / 8;
  } else {
    p.s.passes = (bits + EMB_BITS - 1) / EMB_BITS;
    p.s.bits = (bits + p.s.passes - 1) / p.s.passes;
    const int64_t want = nof_div_up(N, 1024);
    const int64_t per = nof_div_up(N, want < EMB_MAX_BLOCKS ? want : EMB_MAX_BLOCKS);
    p.s.per = (uint32_t)(nof_div_up(per, EMB_SORT_T) * EMB_SORT_T);
    p.s.n_blocks = (int)nof_div_up(N, p.s.per);
  }
  const int64_t nv = nof_div_up(D, 16 / size);
  p.ls = learn_log2_up(nv < EMB_T ? nv : EMB_T);
  p.C = emb_chunk(N, D, size);
  p.chunks = (uint32_t)nof_div_up(N, p.C);
  p.n_red = (uint32_t)nof_div_up(p.chunks, EMB_T >> p.ls);
  int64_t at = 0;
  for (int k = 0; k < 2; ++k) {
    p.key[k] = at; at += learn_align(4 * N);
    p.pos[k] = at; at += learn_align(4 * N);
  }
  p.hist = at; at += learn_align(p.small ? 0 : (int64_t)4 * p.s.n_blocks << p.s.bits);
  p.part = at; at += learn_align((int64_t)p.chunks * 2 * ((D + 7) & ~7) * 4);
  p.bytes = at;
  return p;
}

// whether the sums and the zero role fit a launch (less than 2^32 threads)
static bool emb_launches(const EmbPlan& p) { return (int64_t)p.n_red + EMB_MAX_GRID < (int64_t)1 << 24; }

static bool emb_sizes_ok(int64_t N, int64_t V, int32_t D) {
  return N >= 0 && N < ((int64_t)1 << 31) - 65536 && V >= 0 && V < (int64_t)1 << 30 && D >= 0 && D <= 1 << 20;
}

template <typename T>
static void emb_launch_fwd(const void* table, int64_t stride, const void* ids, int ids64, float scale, void* out, int64_t N, int64_t rows,
                           int32_t D, LearnStream& st) {
  const int64_t nv = nof_div_up(D, EmbVec<T>::V);
  const int ls = learn_log2_up(nv < EMB_T ? nv : EMB_T);
  const int64_t want = nof_div_up(N, EMB_T >> ls), most = (int64_t)1 << 20;
  LEARN_LAUNCH(k_embed_fwd<T>, dim3((unsigned)(want < most ? want : most), (unsigned)nof_div_up(nv, (int64_t)1 << ls)), dim3(EMB_T), 0, st,
                     (const T*)table, stride, ids, ids64, scale, (T*)out, N, rows, D, ls);
}

template <typename T>
static void emb_launch_sums(const void* dout, int64_t stride, const uint32_t* key, const uint32_t* pos, float scale, void* grad, float* part,
                            const EmbPlan& p, int32_t D, LearnStream& st) {
  const unsigned cols = (unsigned)nof_div_up(nof_div_up(D, EmbVec<T>::V), (int64_t)1 << p.ls);
  const int64_t zeros = nof_div_up(p.s.rows - p.zeroed, EMB_ZROWS);
  const unsigned n_zero = (unsigned)(zeros < EMB_MAX_GRID ? zeros : EMB_MAX_GRID);
  // dout past the caches from half of the last one (256 MB) on.  65536 x 2048 bf16: the table's rows stay, a lookup behind it takes 60 us
  // instead of 84; 8192 x 1024: the launch takes 30 us so, 20 through the caches, where dout still lies.
  auto reduce = (int64_t)p.s.N * D * (int64_t)sizeof(T) >= (int64_t)128 << 20 ? k_embed_reduce<T, true> : k_embed_reduce<T, false>;
  LEARN_LAUNCH(reduce, dim3(p.n_red + n_zero, cols), dim3(EMB_T), 0, st, (const T*)dout, stride, key, pos, p.s.N, (uint32_t)p.s.rows, D, scale,
                     (T*)grad, part, p.ls, p.C, p.n_red, (uint32_t)p.zeroed);
  if (p.chunks > 1) {
    const int64_t jv = nof_div_up(D, 4);
    const int jl = learn_log2_up(jv < 64 ? jv : 64);
    LEARN_LAUNCH(k_embed_join<T>, dim3(p.chunks < EMB_MAX_GRID ? p.chunks : EMB_MAX_GRID, (unsigned)nof_div_up(jv, (int64_t)1 << jl)), dim3(EMB_T), 0, st, key, p.s.N,
                       (uint32_t)p.s.rows, D, scale, (T*)grad, (const float*)part, jl, p.C);
  }
}

// at most eight lanes a row, so that a frequent id is many groups' work
template <typename T>
static void emb_launch_few(const void* dout, int64_t stride, const void* ids, int ids64, float scale, void* grad, const EmbPlan& p, int32_t D, LearnStream& st) {
  const int64_t nv = nof_div_up(D, EmbVec<T>::V);
  const int ls = learn_log2_up(nv < 8 ? nv : 8);
  LEARN_LAUNCH(k_embed_few<T>, dim3((unsigned)p.s.rows, (unsigned)nof_div_up(nv, (int64_t)1 << ls)), dim3(EMB_T), 0, st, (const T*)dout, stride, ids,
                     ids64, (int)p.s.N, D, scale, (T*)grad, ls);
}

extern "C" int nof_embed_fwd(const void* table, int64_t table_stride, int32_t type, const void* ids, int32_t ids64, float scale, void* out,
                             int64_t N, int64_t V, int32_t D, void* stream) {
  NOF_ARG(learn_type_ok(type) && (ids64 == 0 || ids64 == 1));
  NOF_ARG(emb_sizes_ok(N, V, D) && table_stride >= 0);
  if (N == 0 || D == 0) return 0;
  NOF_ARG(ids && out && (table || V == 0));
  LearnStream st = {(hipStream_t)stream, hipSuccess};
  if (type == NOF_TYPE_F32) emb_launch_fwd<float>(table, table_stride, ids, ids64, scale, out, N, V, D, st);
  else if (type == NOF_TYPE_BF16) emb_launch_fwd<__bf16>(table, table_stride, ids, ids64, scale, out, N, V, D, st);
  else emb_launch_fwd<_Float16>(table, table_stride, ids, ids64, scale, out, N, V, D, st);
  LEARN_END(st);
  return 0;
}

extern "C" int64_t nof_embed_bwd_workspace_bytes(int64_t N, int64_t V, int32_t D) {
  if (!emb_sizes_ok(N, V, D)) return -1;
  const EmbPlan a = emb_plan(N, V, D, 2), b = emb_plan(N, V, D, 4);    // (of any type)
  if (!emb_launches(a)) return -1;                                    // (wider rows take more)
  return emb_launches(b) && b.bytes > a.bytes ? b.bytes : a.bytes;
}

extern "C" int nof_embed_bwd(const void* dout, int64_t dout_stride, int32_t type, const void* ids, int32_t ids64, float scale,
                             void* grad_table, void* workspace, int64_t workspace_bytes, int64_t N, int64_t V, int32_t D, void* stream) {
  NOF_ARG(learn_type_ok(type) && (ids64 == 0 || ids64 == 1));
  NOF_ARG(emb_sizes_ok(N, V, D) && dout_stride >= 0);
  if (V == 0 || D == 0) return 0;
  NOF_ARG(grad_table && (N == 0 || (dout && ids && workspace)));
  EmbPlan p = emb_plan(N, V, D, (int)learn_type_size(type));
  NOF_ARG(emb_launches(p));
  NOF_ARG(N == 0 || workspace_bytes >= p.bytes);
  NOF_ARG(N == 0 || ((uintptr_t)workspace & 255) == 0);
  LearnStream st = {(hipStream_t)stream, hipSuccess};
  if (p.few) {
    if (type == NOF_TYPE_F32) emb_launch_few<float>(dout, dout_stride, ids, ids64, scale, grad_table, p, D, st);
    else if (type == NOF_TYPE_BF16) emb_launch_few<__bf16>(dout, dout_stride, ids, ids64, scale, grad_table, p, D, st);
    else emb_launch_few<_Float16>(dout, dout_stride, ids, ids64, scale, grad_table, p, D, st);
    LEARN_END(st);
    return 0;
  }
  char* ws = (char*)workspace;
  uint32_t *key[2] = {nullptr, nullptr}, *pos[2] = {nullptr, nullptr};
  float* part = nullptr;
  int cur = 0;
  if (N > 0) {
    for (int k = 0; k < 2; ++k) { key[k] = (uint32_t*)(ws + p.key[k]); pos[k] = (uint32_t*)(ws + p.pos[k]); }
    part = (float*)(ws + p.part);
    uint32_t* hist = (uint32_t*)(ws + p.hist);
    p.s.ids = ids;
    p.s.ids64 = ids64;
    // what the launches of the sort have time for
    const int64_t row = D * learn_type_size(type), room = p.small ? EMB_ZSMALL : p.s.passes * (EMB_ZHIST + EMB_ZSCATTER);
    p.zeroed = room / row < V ? room / row : V;
    EmbZero z = {(char*)grad_table, 0};
    int64_t left = p.zeroed * row;
    auto share = [&](int64_t most) {                                  // the next stretch; its workgroups
      z.at += z.bytes;
      z.bytes = (uint64_t)(left < most ? left : most);
      left -= (int64_t)z.bytes;
      return (unsigned)nof_div_up((int64_t)z.bytes, EMB_ZBYTES);
    };
    if (p.small) {
      const unsigned more = share(left);
      LEARN_LAUNCH(k_embed_sort_small, dim3(1 + more), dim3(1024), 0, st, ids, (int)ids64, V, (int)N, p.s.passes, key[0], pos[0], z);
    } else {
      for (int pass = 0; pass < p.s.passes; ++pass, cur ^= 1) {
        unsigned more = share(EMB_ZHIST);
        LEARN_LAUNCH(k_embed_hist, dim3(p.s.n_blocks + more), dim3(EMB_SORT_T), 0, st, p.s, pass, (const uint32_t*)key[cur], hist, z);
        more = share(EMB_ZSCATTER);
        LEARN_LAUNCH(k_embed_scatter, dim3(p.s.n_blocks + more), dim3(EMB_SORT_T), 0, st, p.s, pass, (const uint32_t*)key[cur],
                           (const uint32_t*)pos[cur], key[cur ^ 1], pos[cur ^ 1], (const uint32_t*)hist, z);
      }
    }
    LEARN_END(st);
  }
  if (type == NOF_TYPE_F32) emb_launch_sums<float>(dout, dout_stride, key[cur], pos[cur], scale, grad_table, part, p, D, st);
  else if (type == NOF_TYPE_BF16) emb_launch_sums<__bf16>(dout, dout_stride, key[cur], pos[cur], scale, grad_table, part, p, D, st);
  else emb_launch_sums<_Float16>(dout, dout_stride, key[cur], pos[cur], scale, grad_table, part, p, D, st);
  LEARN_END(st);
  return 0;
}
