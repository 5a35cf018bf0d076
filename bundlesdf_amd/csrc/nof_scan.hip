// Gated linear recurrence along time with its backward pass and its single step (nof_gated_scan_*, include/nof_hip.h).
//
//   forward    h[t] = a[t] h[t-1] + x[t],  h[-1] = state               a: the gate, one per channel or one per group of P = D / G channels
//   backward   r[t] = dh[t] + a[t+1] r[t+1]  (the last position adds dlast)
//              dx[t] = r[t],  da[t] = sum over the group of r[t] h[t-1],  dstate = a[0] r[0]
//
// Bound by memory: the forward reads a, x and writes h once, the backward reads a, x, dh and writes da, dx.  Composition of two steps
// (a, b) then (a', b') is (a a', a' b + b'), so time is cut: a workgroup of up to four waves takes a CHUNK of positions at a time, each of its
// slots SCAN_U consecutive positions of one lane's channels in registers (as loaded; converted where used); slots compose their (a, b) by
// shuffles within a wave and through LDS between waves -- one barrier a chunk --, the state between chunks stays in registers.  Three such
// workgroups a compute unit (two in the backward of a shared gate's pairs) hide each other's loads.  Where batch x channels give too few workgroups, time is also cut into segments: a first
// launch composes each segment (its slots walk their share without a barrier), and every workgroup of the second folds the segments before
// its own.
//
// The backward needs h[t-1] in binary32, not as the output rounded it: the forward leaves the state in front of every chunk of the backward
// ("marks", 4 / chunk bytes per element), and the backward runs the chunk forward again from there.  Rounded states instead would cost the
// gate's gradient up to half a step of the value's type.
//
// Lanes hold tiles of CT = 2^cs channels (V each); 64 / CT positions side by side fill a wave where channels are few.  In the backward a tile
// never spans two groups of a shared gate, so the gate's gradient is one sum over the tile's lanes; a group of several tiles adds them in a
// second launch, in order.
#include "nof_learn_dev.h"
#include <type_traits>

#define SCAN_U 16
#define SCAN_MAXW 4                     // waves per workgroup at most

struct ScanArgs {
  const void* gate; const void* value; const void* dh;
  int64_t gate_sb, gate_st, value_sb, value_st, dh_sb, dh_st;        // elements between batches and positions
  const float* state;                   // [B, D] or NULL
  const int32_t* lengths;               // [B] or NULL
  void* h; float* last; float* marks;
  const float* dlast;
  void* dvalue; void* dgate; float* dstate; float* gpart;
  float* seg;                           // segment summaries [segs][B][2][D]
  int64_t T;
  int B, D, G, P;                       // P = channels per gate
  int per_channel, reverse;
  int mark, n_marks;                    // positions between marks (the backward's chunk)
  // the layout of a launch
  int span;                             // channels that a row of tiles covers: D, or P where tiles keep to a gate's group
  int cs, tiles_per_span, tiles;
  int waves, chunk, n_chunks, segs, chunks_per_seg;
};

__device__ __forceinline__ int64_t scan_len(const ScanArgs& p, int b) {
  if (!p.lengths) return p.T;
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : n > p.T ? p.T : n;
}

struct ScanWhere { int b, ch, span, slot; bool on; int64_t n; };

// this thread's channels (an idle lane of a ragged tile reads its span's first ones and stores nothing) and its slot
template <int V>
__device__ __forceinline__ ScanWhere scan_where(const ScanArgs& p) {
  ScanWhere q;
  const int lane = threadIdx.x & 63, ct = 1 << p.cs, tile = blockIdx.x % p.tiles;
  q.b = blockIdx.x / p.tiles;
  q.span = tile / p.tiles_per_span;
  const int in_span = ((tile % p.tiles_per_span) * ct + (lane & (ct - 1))) * V;
  q.on = in_span < p.span;
  q.ch = q.span * p.span + (q.on ? in_span : 0);
  q.slot = (threadIdx.x >> 6) * (64 >> p.cs) + (lane >> p.cs);
  q.n = scan_len(p, q.b);
  return q;
}

// rows of one lane's channels in the recurrence's order: position i of the tensor's n existing rows
template <typename T> struct ScanRows {
  T* base; int64_t step;
  __device__ __forceinline__ ScanRows(T* first, int64_t st, const ScanArgs& p, int64_t n) : base(p.reverse ? first + (n - 1) * st : first), step(p.reverse ? -st : st) {}
  __device__ __forceinline__ T* at(int64_t i) const { return base + i * step; }
  // the step for a run of rows.  (No instruction: the rows' offsets are formed at the run; hoisted before the chunks they fill the scalar
  // registers and spill.)
  __device__ __forceinline__ int64_t stride() const {
    int64_t s = step;
    asm volatile("" : "+s"(s));
    return s;
  }
};

// V elements as they lie in memory, two 16-bit ones in one register (as elements, the compiler gives each a register of its own and spills)
template <int BYTES> struct ScanBits;
template <> struct ScanBits<2> { typedef uint16_t t; };
template <> struct ScanBits<4> { typedef uint32_t t; };
template <> struct ScanBits<8> { typedef uint2 t; };
template <typename T, int V> using ScanRaw = typename ScanBits<sizeof(T) * V>::t;
__device__ __forceinline__ float scan_16(uint16_t b, __bf16) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ float scan_16(uint16_t b, _Float16) { return (float)__builtin_bit_cast(_Float16, b); }
__device__ __forceinline__ float scan_16(uint16_t b, float) { return 0.0f; }
template <typename T, int V> __device__ __forceinline__ float scan_get(const ScanRaw<T, V>& r, int v) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 2) return __uint_as_float(v ? r.y : r.x);
    else return __uint_as_float(r);
  } else if constexpr (V == 2) {
    return scan_16((uint16_t)(v ? r >> 16 : r & 0xffffu), T());
  } else {
    return scan_16(r, T());
  }
}
template <typename T, int V> __device__ __forceinline__ ScanRaw<T, V> scan_fill(float x) {
  LearnVec<T, V> f;
#pragma unroll
  for (int v = 0; v < V; ++v) f.v[v] = lt<T>(x);
  return __builtin_bit_cast(ScanRaw<T, V>, f);
}

// SCAN_U positions from i0 on of n > 0; positions from n on are `fill` (their loads go to the last row: a branch per row, or a predicate
// per row and array, costs the compiler its registers).  The choice is each slot's: made for a whole segment, 24 x 1777 x 520 of uneven
// lengths took 18 us to compose, 12 so.
template <typename T, int V>
__device__ __forceinline__ void scan_fetch(const ScanRows<const T>& x, int64_t i0, int64_t n, float fill, ScanRaw<T, V> (&r)[SCAN_U]) {
  const T* p = x.at(i0);
  const int64_t st = x.stride(), left = n - i0;
  if (left >= SCAN_U) {
#pragma unroll
    for (int u = 0; u < SCAN_U; ++u) r[u] = *reinterpret_cast<const ScanRaw<T, V>*>(p + u * st);
  } else {
#pragma unroll
    for (int u = 0; u < SCAN_U; ++u) {
      const ScanRaw<T, V> in = *reinterpret_cast<const ScanRaw<T, V>*>(p + (u < left ? u : left - 1) * st), out = scan_fill<T, V>(fill);
      r[u] = u < left ? in : out;
    }
  }
}

// Composition over the slots of a workgroup, in slot order (REV: from the last slot down), in three parts so that two directions share a
// barrier.  scan_wave: (A, B) of this slot -> of the slots before it in its wave, and the wave's whole into `sh`.
template <int V, bool REV>
__device__ __forceinline__ void scan_wave(float (&A)[V], float (&B)[V], int cs, float2* sh) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, ct = 1 << cs, sub = lane >> cs, nsub = 64 >> cs, at = REV ? nsub - 1 - sub : sub;
  for (int o = 1; o < nsub; o <<= 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float a = REV ? __shfl_down(A[v], o * ct) : __shfl_up(A[v], o * ct), b = REV ? __shfl_down(B[v], o * ct) : __shfl_up(B[v], o * ct);
      if (at >= o) { B[v] = A[v] * b + B[v]; A[v] *= a; }
    }
  }
  if (at == nsub - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) sh[(w * V + v) * 64 + (lane & (ct - 1))] = make_float2(A[v], B[v]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float a = nsub == 1 ? 1.0f : REV ? __shfl_down(A[v], ct) : __shfl_up(A[v], ct);
    const float b = nsub == 1 ? 0.0f : REV ? __shfl_down(B[v], ct) : __shfl_up(B[v], ct);
    A[v] = at > 0 ? a : 1.0f;
    B[v] = at > 0 ? b : 0.0f;
  }
}
// behind a barrier: (A, B) -> of all slots before this one, (TA, TB) = of all slots
template <int V, bool REV>
__device__ __forceinline__ void scan_fold(float (&A)[V], float (&B)[V], float (&TA)[V], float (&TB)[V], int cs, int waves, const float2* sh) {
  const int l = threadIdx.x & ((1 << cs) - 1), w = threadIdx.x >> 6;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float pa = 1.0f, pb = 0.0f;
    TA[v] = 1.0f;
    TB[v] = 0.0f;
#pragma unroll
    for (int k = 0; k < SCAN_MAXW; ++k) {
      const int q = REV ? SCAN_MAXW - 1 - k : k;
      if (q < waves) {
        if (q == w) { pa = TA[v]; pb = TB[v]; }
        const float2 s = sh[(q * V + v) * 64 + l];
        TB[v] = s.x * TB[v] + s.y;
        TA[v] *= s.x;
      }
    }
    B[v] = A[v] * pb + B[v];
    A[v] *= pa;
  }
}

// The composition of a whole segment.  BACK: of the recurrence of what positions hand to the one before, c[t-1] = a[t] (dh[t] + c[t]).
// The segment's slots take equal stretches of it, so that the only barrier is the last composition's.
template <typename TG, typename T, int V, bool PC, bool BACK>
__global__ __launch_bounds__(64 * SCAN_MAXW, PC && V == 2 && sizeof(TG) == 4 ? 3 : 4) void k_scan_segments(ScanArgs p) {
  __shared__ float2 sh[SCAN_MAXW * 64 * V];
  const ScanWhere q = scan_where<V>(p);
  const int seg = BACK ? blockIdx.y + 1 : blockIdx.y;               // nobody needs the forward's last or the backward's first
  const ScanRows<const TG> g((const TG*)p.gate + q.b * p.gate_sb + (PC ? q.ch : q.ch / p.P), p.gate_st, p, q.n);
  const ScanRows<const T> x(BACK ? (const T*)p.dh + q.b * p.dh_sb + q.ch : (const T*)p.value + q.b * p.value_sb + q.ch, BACK ? p.dh_st : p.value_st, p, q.n);
  const int64_t seg0 = (int64_t)seg * p.chunks_per_seg * p.chunk, each = (int64_t)p.chunks_per_seg * SCAN_U, i0 = seg0 + q.slot * each;
  float A[V], B[V], TA[V], TB[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { A[v] = 1.0f; B[v] = 0.0f; }
  // two runs of positions in turn, the next one's loads under way while one is composed
  ScanRaw<TG, PC ? V : 1> a[2][SCAN_U];
  ScanRaw<T, V> r[2][SCAN_U];
  auto place = [&](int k) { return i0 + (int64_t)(BACK ? p.chunks_per_seg - 1 - k : k) * SCAN_U; };
  auto fetch = [&](int k, auto& to, auto& too) {
    const int64_t i = place(k);
    if (k < p.chunks_per_seg && i < q.n) {
      scan_fetch<TG, PC ? V : 1>(g, i, q.n, 1.0f, to);
      scan_fetch<T, V>(x, i, q.n, 0.0f, too);
    }
  };
  auto compose = [&](int k, const auto& a, const auto& r) {
    if (k >= p.chunks_per_seg || place(k) >= q.n) return;
#pragma unroll
    for (int t = 0; t < SCAN_U; ++t) {
      const int u = BACK ? SCAN_U - 1 - t : t;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float av = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0), xv = scan_get<T, V>(r[u], v);
        B[v] = BACK ? av * (xv + B[v]) : av * B[v] + xv;
        A[v] *= av;
      }
    }
  };
  fetch(0, a[0], r[0]);
  for (int k = 0; k < p.chunks_per_seg; k += 2) {
    fetch(k + 1, a[1], r[1]);
    compose(k, a[0], r[0]);
    fetch(k + 2, a[0], r[0]);
    compose(k + 1, a[1], r[1]);
  }
  scan_wave<V, BACK>(A, B, p.cs, sh);
  __syncthreads();
  scan_fold<V, BACK>(A, B, TA, TB, p.cs, p.waves, sh);
  if (q.slot == 0 && q.on) {
    float* out = p.seg + (((int64_t)seg * p.B + q.b) * 2) * p.D + q.ch;
    lstore<float, V>(out, TA);
    lstore<float, V>(out + p.D, TB);
  }
}

// S -> what it becomes over segments lo, lo + step, ... (count of them).  Many of them are composed by the workgroup's slots, a stretch each:
// one slot's walk over 511 segments is a chain of 511 loads (1 x 65536 x 64 fp32 forward: 49 us so, 22 by slots).
template <int V>
__device__ __forceinline__ void scan_over(const ScanArgs& p, const ScanWhere& q, int lo, int step, int count, float (&S)[V], float2* sh) {
  const bool share = count > 16;
  const int slots = p.waves * (64 >> p.cs), each = share ? (count + slots - 1) / slots : count;
  const int k0 = share ? q.slot * each : 0, k1 = k0 + each < count ? k0 + each : count;
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { A[v] = 1.0f; B[v] = 0.0f; }
#pragma unroll 8
  for (int k = k0; k < k1; ++k) {
    float a[V], b[V];
    const float* s = p.seg + (((int64_t)(lo + k * step) * p.B + q.b) * 2) * p.D + q.ch;
    lload<float, V>(s, a);
    lload<float, V>(s + p.D, b);
#pragma unroll
    for (int v = 0; v < V; ++v) { B[v] = a[v] * B[v] + b[v]; A[v] *= a[v]; }
  }
  if (share) {
    float TA[V], TB[V];
    scan_wave<V, false>(A, B, p.cs, sh);
    __syncthreads();
    scan_fold<V, false>(A, B, TA, TB, p.cs, p.waves, sh);
    __syncthreads();                                                  // (sh is the chunks' next)
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = TA[v]; B[v] = TB[v]; }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) S[v] = A[v] * S[v] + B[v];
}

template <typename TG, typename T, int V, bool PC>
__global__ __launch_bounds__(64 * SCAN_MAXW, 3) void k_scan_fwd(ScanArgs p) {
  __shared__ float2 sh[2][SCAN_MAXW * 64 * V];
  const ScanWhere q = scan_where<V>(p);
  const ScanRows<const TG> g((const TG*)p.gate + q.b * p.gate_sb + (PC ? q.ch : q.ch / p.P), p.gate_st, p, q.n);
  const ScanRows<const T> x((const T*)p.value + q.b * p.value_sb + q.ch, p.value_st, p, q.n);
  T* h0 = p.h ? (T*)p.h + (int64_t)q.b * p.T * p.D + q.ch : nullptr;
  const ScanRows<T> h(h0, p.D, p, q.n);
  const int seg = blockIdx.y, c0 = seg * p.chunks_per_seg, c1 = c0 + p.chunks_per_seg < p.n_chunks ? c0 + p.chunks_per_seg : p.n_chunks;
  float S[V];
#pragma unroll
  for (int v = 0; v < V; ++v) S[v] = 0.0f;
  if (p.state) lload<float, V>(p.state + (int64_t)q.b * p.D + q.ch, S);
  ScanRaw<TG, PC ? V : 1> a[SCAN_U];
  ScanRaw<T, V> r[SCAN_U];
  const int64_t at0 = (int64_t)c0 * p.chunk;
  if (at0 < q.n) {
    scan_fetch<TG, PC ? V : 1>(g, at0 + q.slot * SCAN_U, q.n, 1.0f, a);
    scan_fetch<T, V>(x, at0 + q.slot * SCAN_U, q.n, 0.0f, r);
  }
  scan_over<V>(p, q, 0, 1, seg, S, sh[0]);
  for (int c = c0; c < c1; ++c) {
    const int64_t at = (int64_t)c * p.chunk, i0 = at + q.slot * SCAN_U;
    const bool full = i0 + SCAN_U <= q.n;
    if (at < q.n) {
      float A[V], B[V], TA[V], TB[V], s[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { A[v] = 1.0f; B[v] = 0.0f; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) { const float av = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0); B[v] = av * B[v] + scan_get<T, V>(r[u], v); A[v] *= av; }
      scan_wave<V, false>(A, B, p.cs, sh[c & 1]);
      __syncthreads();
      scan_fold<V, false>(A, B, TA, TB, p.cs, p.waves, sh[c & 1]);
#pragma unroll
      for (int v = 0; v < V; ++v) { s[v] = A[v] * S[v] + B[v]; S[v] = TA[v] * S[v] + TB[v]; }
      if (p.marks && q.on && i0 < q.n && (uint32_t)i0 % (uint32_t)p.mark == 0)
        lstore<float, V>(p.marks + ((int64_t)q.b * p.n_marks + (uint32_t)i0 / (uint32_t)p.mark) * p.D + q.ch, s);
      T* o = h.at(i0);
      const int64_t ost = h.stride();
      const int64_t left = q.n - i0;
      auto run = [&](auto whole) {
#pragma unroll
        for (int u = 0; u < SCAN_U; ++u) {
#pragma unroll
          for (int v = 0; v < V; ++v) s[v] = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0) * s[v] + scan_get<T, V>(r[u], v);
          if (whole.value || u < left) lstore<T, V>(o + u * ost, s);
        }
      };
      if (q.on && h0) {                                               // (one branch, not one per row)
        if (full) run(std::true_type()); else run(std::false_type());
      } else {
#pragma unroll
        for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
          for (int v = 0; v < V; ++v) s[v] = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0) * s[v] + scan_get<T, V>(r[u], v);
      }
      // (positions behind the end keep the state)
      if (p.last && q.on && i0 < q.n && i0 + SCAN_U >= q.n) lstore<float, V>(p.last + (int64_t)q.b * p.D + q.ch, s);
      if (c + 1 < c1 && at + p.chunk < q.n) {
        scan_fetch<TG, PC ? V : 1>(g, i0 + p.chunk, q.n, 1.0f, a);
        scan_fetch<T, V>(x, i0 + p.chunk, q.n, 0.0f, r);
      }
    }
    if (h0 && q.on && !full) {                                        // rows behind the sequence's end
      float z[V];
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = 0.0f;
      for (int64_t i = i0 > q.n ? i0 : q.n; i < i0 + SCAN_U && i < p.T; ++i) lstore<T, V>(h0 + i * p.D, z);
    }
  }
  if (q.n == 0 && seg == 0 && q.slot == 0 && q.on && p.last) lstore<float, V>(p.last + (int64_t)q.b * p.D + q.ch, S);
}

// sum of f[u] over the 2^cs lanes of a tile, for all SCAN_U values: each exchange halves what is left to add, so 16 values over 64 lanes
// take 8 + 4 + 2 + 1 + 2 exchanges instead of 96.  The highest bits of a lane's index in the tile choose between the upper and the
// lower half of what was left; lanes that agree in them end with the same sums f[0 .. left).
__device__ __forceinline__ void scan_tile_sum(float (&f)[SCAN_U], int cs) {
  const int lane = threadIdx.x & 63;
  int left = SCAN_U;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    if (k >= cs) break;
    const int o = 1 << (cs - 1 - k);
    if (left > 1) {
      left >>= 1;
      const bool upper = lane & o;
#pragma unroll
      for (int j = 0; j < SCAN_U / 2; ++j)
        if (j < left) {
          const float mine = upper ? f[j + left] : f[j], other = upper ? f[j] : f[j + left];
          f[j] = mine + __shfl_xor(other, o);
        }
    } else {
      f[0] += __shfl_xor(f[0], o);
    }
  }
}

template <typename TG, typename T, int V, bool PC>
__global__ __launch_bounds__(64 * SCAN_MAXW, PC || V == 1 ? 3 : 2) void k_scan_bwd(ScanArgs p) {
  __shared__ float2 sh[2][2][SCAN_MAXW * 64 * V];
  const ScanWhere q = scan_where<V>(p);
  const int lane = threadIdx.x & 63, ct = 1 << p.cs, part = blockIdx.x % p.tiles % p.tiles_per_span, group = PC ? 0 : q.span;
  const ScanRows<const TG> g((const TG*)p.gate + q.b * p.gate_sb + (PC ? q.ch : group), p.gate_st, p, q.n);
  const ScanRows<const T> x((const T*)p.value + q.b * p.value_sb + q.ch, p.value_st, p, q.n), y((const T*)p.dh + q.b * p.dh_sb + q.ch, p.dh_st, p, q.n);
  T* dx0 = (T*)p.dvalue + (int64_t)q.b * p.T * p.D + q.ch;
  const ScanRows<T> dx(dx0, p.D, p, q.n);
  TG* dg0 = PC ? (TG*)p.dgate + (int64_t)q.b * p.T * p.D + q.ch : (TG*)p.dgate + (int64_t)q.b * p.T * p.G + group;
  const ScanRows<TG> dg(dg0, PC ? p.D : p.G, p, q.n);
  float* gp0 = p.gpart + ((int64_t)q.b * p.T * p.G + group) * p.tiles_per_span + part;               // (a shared gate of several tiles)
  const ScanRows<float> gp(gp0, (int64_t)p.G * p.tiles_per_span, p, q.n);
  const int seg = blockIdx.y, c0 = seg * p.chunks_per_seg, c1 = c0 + p.chunks_per_seg < p.n_chunks ? c0 + p.chunks_per_seg : p.n_chunks;
  float R[V];                                                       // what later positions hand to this one
#pragma unroll
  for (int v = 0; v < V; ++v) R[v] = 0.0f;
  if (p.dlast) lload<float, V>(p.dlast + (int64_t)q.b * p.D + q.ch, R);
  scan_over<V>(p, q, p.segs - 1, -1, p.segs - 1 - seg, R, sh[0][0]);
  for (int c = c1 - 1; c >= c0; --c) {
    const int64_t at = (int64_t)c * p.chunk, i0 = at + q.slot * SCAN_U;
    const bool full = i0 + SCAN_U <= q.n;
    if (at < q.n) {
      ScanRaw<TG, PC ? V : 1> a[SCAN_U];
      ScanRaw<T, V> r[SCAN_U], d[SCAN_U];
      float A[V], B[V], A2[V], B2[V], TA[V], TB[V], m[V], s[V], hp[SCAN_U][V];
      scan_fetch<TG, PC ? V : 1>(g, i0, q.n, 1.0f, a);
      scan_fetch<T, V>(x, i0, q.n, 0.0f, r);
      scan_fetch<T, V>(y, i0, q.n, 0.0f, d);
      lload<float, V>(p.marks + ((int64_t)q.b * p.n_marks + c) * p.D + q.ch, m);
#pragma unroll
      for (int v = 0; v < V; ++v) { A[v] = 1.0f; B[v] = 0.0f; B2[v] = 0.0f; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) { const float av = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0); B[v] = av * B[v] + scan_get<T, V>(r[u], v); A[v] *= av; }
#pragma unroll
      for (int u = SCAN_U - 1; u >= 0; --u)
#pragma unroll
        for (int v = 0; v < V; ++v) B2[v] = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0) * (scan_get<T, V>(d[u], v) + B2[v]);
#pragma unroll
      for (int v = 0; v < V; ++v) A2[v] = A[v];
      scan_wave<V, false>(A, B, p.cs, sh[c & 1][0]);
      scan_wave<V, true>(A2, B2, p.cs, sh[c & 1][1]);
      __syncthreads();
      scan_fold<V, false>(A, B, TA, TB, p.cs, p.waves, sh[c & 1][0]);
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = A[v] * m[v] + B[v];
      scan_fold<V, true>(A2, B2, TA, TB, p.cs, p.waves, sh[c & 1][1]);
#pragma unroll
      for (int v = 0; v < V; ++v) { B2[v] = A2[v] * R[v] + B2[v]; R[v] = TA[v] * R[v] + TB[v]; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) { hp[u][v] = s[v]; s[v] = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0) * s[v] + scan_get<T, V>(r[u], v); }
      T* o = dx.at(i0);
      TG* og = dg.at(i0);
      const int64_t ost = dx.stride(), gst = dg.stride();
      float f[SCAN_U];
      const int64_t left = q.n - i0;
      auto run = [&](auto whole) {
#pragma unroll
        for (int u = SCAN_U - 1; u >= 0; --u) {
          float e[V];
          f[u] = 0.0f;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            e[v] = scan_get<T, V>(d[u], v) + B2[v];                   // r[t]
            hp[u][v] *= e[v];
            B2[v] = scan_get<TG, PC ? V : 1>(a[u], PC ? v : 0) * e[v];
            f[u] += hp[u][v];
          }
          if (whole.value || u < left) {
            lstore<T, V>(o + u * ost, e);
            if (PC) lstore<TG, V>(og + u * gst, hp[u]);
          }
        }
      };
      if (q.on) {                                                     // (one branch, not one per row)
        if (full) run(std::true_type()); else run(std::false_type());
      } else {
#pragma unroll
        for (int u = 0; u < SCAN_U; ++u) f[u] = 0.0f;
      }
      if (!PC) {
        scan_tile_sum(f, p.cs);
        const int in = lane & (ct - 1);
        int mine = SCAN_U, u0 = 0;
        for (int k = 0; k < 4 && k < p.cs; ++k) { mine >>= 1; if (in >> (p.cs - 1 - k) & 1) u0 += mine; }
        const int low = p.cs > 4 ? in & ((1 << (p.cs - 4)) - 1) : 0;
#pragma unroll
        for (int j = 0; j < SCAN_U; ++j)
          if (low == 0 && j < mine && u0 + j < left) {
            if (p.tiles_per_span == 1) *dg.at(i0 + u0 + j) = lt<TG>(f[j]);
            else *gp.at(i0 + u0 + j) = f[j];
          }
      }
    }
    if (q.on && !full) {                                              // rows behind the sequence's end have no gradient
      float z[V];
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = 0.0f;
      for (int64_t i = i0 > q.n ? i0 : q.n; i < i0 + SCAN_U && i < p.T; ++i) {
        lstore<T, V>(dx0 + i * p.D, z);
        if (PC) lstore<TG, V>(dg0 + i * p.D, z);
        else if ((lane & (ct - 1)) == 0) {
          if (p.tiles_per_span == 1) dg0[i * p.G] = lt<TG>(0.0f);
          else gp0[i * p.G * p.tiles_per_span] = 0.0f;
        }
      }
    }
  }
  if (seg == 0 && q.slot == 0 && q.on && p.dstate) lstore<float, V>(p.dstate + (int64_t)q.b * p.D + q.ch, R);
}

// the tiles of a shared gate's group, added in order
template <typename TG>
__global__ __launch_bounds__(256) void k_scan_gate_sum(const float* __restrict__ gpart, TG* __restrict__ dgate, int64_t n, int k) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.0f;
    for (int j = 0; j < k; ++j) s += gpart[i * k + j];
    dgate[i] = lt<TG>(s);
  }
}

// (new_state may be what a lane has read: its own elements of state, or of a float32 gate or value)
template <typename TG, typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(const TG* gate, int64_t gate_st, const T* value, int64_t value_st, const float* state,
                                                   float* new_state, T* __restrict__ h, int B, int D, int G, int blocks_per_row) {
  const int b = blockIdx.x / blocks_per_row, ch = ((blockIdx.x % blocks_per_row) * 256 + threadIdx.x) * V;
  if (ch >= D) return;
  float a[V], x[V], s[V];
  if (G == D) lload<TG, V>(gate + b * gate_st + ch, a);
  else {
    const float one = lf(gate[b * gate_st + ch / (D / G)]);            // V divides D / G: one group a lane
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = one;
  }
  lload<T, V>(value + b * value_st + ch, x);
  lload<float, V>(state + (int64_t)b * D + ch, s);
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = a[v] * s[v] + x[v];
  lstore<float, V>(new_state + (int64_t)b * D + ch, s);
  lstore<T, V>(h + (int64_t)b * D + ch, s);
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
// Everything here depends on the sizes alone, so that the forward's marks fit the backward.
// Segments: from one wave per SIMD (1024 waves) on, a workgroup's own look-ahead keeps the memory busy and a second pass over the inputs
// would cost more than it gives; below, two waves per SIMD, of two chunks at least.  4 x 16384 x 1024 bf16, forward + backward: 118 + 177 us
// so, 128 + 198 with four waves per SIMD, 159 + 209 with one.
// Tiles narrower than a wave where that leaves a fifth fewer lanes without a channel: 65 channels a group (24 x 1777 x 520, eight gates)
// backward 84 us, 115 as 64 + 1.
static void scan_layout(ScanArgs& p, int span, int v) {
  p.span = span;
  const int nv = span / v;
  p.cs = learn_log2_up(nv < 64 ? nv : 64);
  for (int cs = 5; nv > 64 && cs >= 4; --cs)                          // (one tile a span stays one: another means sums to join)
    if (5 * (nof_div_up(nv, (int64_t)1 << cs) << cs) <= 4 * (nof_div_up(nv, (int64_t)1 << p.cs) << p.cs)) p.cs = cs;
  p.tiles_per_span = (int)nof_div_up(nv, (int64_t)1 << p.cs);
  p.tiles = p.D / span * p.tiles_per_span;
  const int64_t slots = nof_div_up(p.T, SCAN_U), per_wave = 64 >> p.cs, need = nof_div_up(slots, per_wave);
  p.waves = (int)(need < 1 ? 1 : need < SCAN_MAXW ? need : SCAN_MAXW);
  p.chunk = (int)(p.waves * per_wave * SCAN_U);
  p.n_chunks = (int)nof_div_up(p.T, p.chunk);
  const int64_t waves = (int64_t)p.B * p.tiles * p.waves, want = waves >= 1024 ? 1 : nof_div_up(2048, waves), most = p.n_chunks / 2 > 1 ? p.n_chunks / 2 : 1;
  p.segs = (int)(want < most ? want : most);
  p.chunks_per_seg = (int)nof_div_up(p.n_chunks > 0 ? p.n_chunks : 1, p.segs);
  p.segs = (int)nof_div_up(p.n_chunks > 0 ? p.n_chunks : 1, p.chunks_per_seg);
}
static bool scan_plan(ScanArgs& p, int64_t B, int64_t T, int32_t D, int32_t G, int v, bool back) {
  p.T = T; p.B = (int)B; p.D = D; p.G = G;
  p.per_channel = G == D;
  p.P = D / G;
  scan_layout(p, p.per_channel ? D : p.P, v);
  p.mark = p.chunk;
  p.n_marks = p.n_chunks;
  if (!back) scan_layout(p, D, v);
  return B * p.tiles * p.waves * 64 < (int64_t)1 << 32;               // (threads of a launch)
}

// two 16-bit channels a lane where a group is even
static int scan_vec(int32_t type, int32_t D, int32_t G) {
  const int32_t P = G == D ? D : D / G;
  return type != NOF_TYPE_F32 && P % 2 == 0 ? 2 : 1;
}

static bool scan_sizes_ok(int64_t B, int64_t T, int32_t D, int32_t G) {
  return B >= 0 && B < (int64_t)1 << 24 && T >= 0 && T < (int64_t)1 << 31 && D >= 0 && D <= 1 << 20 && (D == 0 || (G > 0 && G <= D && D % G == 0));
}
static bool scan_types_ok(int32_t type, int32_t gate_type) {
  return learn_type_ok(type) && (gate_type == type || gate_type == NOF_TYPE_F32);
}
static bool scan_aligned(const void* x, int64_t sb, int64_t st, int size, int v) {
  return ((uintptr_t)x % (uintptr_t)(size * v)) == 0 && sb % v == 0 && st % v == 0;
}

#define SCAN_GO(KERNEL, GRID, BLOCK, TG, T, V, ...)                                                          \
  do {                                                                                                       \
    if (p.per_channel) LEARN_LAUNCH((KERNEL<TG, T, V, true, ##__VA_ARGS__>), GRID, BLOCK, 0, st, p);      \
    else LEARN_LAUNCH((KERNEL<TG, T, V, false, ##__VA_ARGS__>), GRID, BLOCK, 0, st, p);                   \
  } while (0)
#define SCAN_PICK(KERNEL, GRID, BLOCK, ...)                                                                  \
  do {                                                                                                       \
    if (type == NOF_TYPE_F32) SCAN_GO(KERNEL, GRID, BLOCK, float, float, 1, ##__VA_ARGS__);                    \
    else if (type == NOF_TYPE_BF16 && gate_type == type) {                                                   \
      if (v == 2) SCAN_GO(KERNEL, GRID, BLOCK, __bf16, __bf16, 2, ##__VA_ARGS__);                              \
      else SCAN_GO(KERNEL, GRID, BLOCK, __bf16, __bf16, 1, ##__VA_ARGS__);                                     \
    } else if (type == NOF_TYPE_BF16) {                                                                      \
      if (v == 2) SCAN_GO(KERNEL, GRID, BLOCK, float, __bf16, 2, ##__VA_ARGS__);                               \
      else SCAN_GO(KERNEL, GRID, BLOCK, float, __bf16, 1, ##__VA_ARGS__);                                      \
    } else if (gate_type == type) {                                                                          \
      if (v == 2) SCAN_GO(KERNEL, GRID, BLOCK, _Float16, _Float16, 2, ##__VA_ARGS__);                          \
      else SCAN_GO(KERNEL, GRID, BLOCK, _Float16, _Float16, 1, ##__VA_ARGS__);                                 \
    } else {                                                                                                 \
      if (v == 2) SCAN_GO(KERNEL, GRID, BLOCK, float, _Float16, 2, ##__VA_ARGS__);                             \
      else SCAN_GO(KERNEL, GRID, BLOCK, float, _Float16, 1, ##__VA_ARGS__);                                    \
    }                                                                                                        \
  } while (0)

static int64_t scan_seg_bytes(const ScanArgs& p) { return p.segs > 1 ? learn_align((int64_t)p.segs * p.B * 2 * p.D * 4) : 0; }
static int64_t scan_gpart_bytes(const ScanArgs& p) {
  return !p.per_channel && p.tiles_per_span > 1 ? learn_align((int64_t)p.B * p.T * p.G * p.tiles_per_span * 4) : 0;
}

extern "C" int64_t nof_gated_scan_marks_bytes(int64_t B, int64_t T, int32_t D, int32_t G, int32_t type) {
  if (!scan_sizes_ok(B, T, D, G) || !learn_type_ok(type)) return -1;
  if (B == 0 || D == 0) return 0;
  ScanArgs p = {};
  if (!scan_plan(p, B, T, D, G, scan_vec(type, D, G), false)) return -1;
  return (int64_t)p.B * p.n_marks * p.D * 4;
}

extern "C" int64_t nof_gated_scan_workspace_bytes(int64_t B, int64_t T, int32_t D, int32_t G, int32_t type) {
  if (!scan_sizes_ok(B, T, D, G) || !learn_type_ok(type)) return -1;
  if (B == 0 || D == 0) return 0;
  ScanArgs p = {};
  if (!scan_plan(p, B, T, D, G, scan_vec(type, D, G), false)) return -1;
  const int64_t fwd = scan_seg_bytes(p);
  if (!scan_plan(p, B, T, D, G, scan_vec(type, D, G), true)) return fwd;                 // (a backward call of these sizes is refused)
  const int64_t bwd = scan_seg_bytes(p) + scan_gpart_bytes(p);
  return fwd > bwd ? fwd : bwd;
}

extern "C" int nof_gated_scan_fwd(const void* gate, int64_t gate_sb, int64_t gate_st, int32_t gate_type, const void* value, int64_t value_sb,
                                  int64_t value_st, int32_t type, const float* state, const int32_t* lengths, int32_t reverse, void* h,
                                  float* last, float* marks, void* workspace, int64_t workspace_bytes, int64_t B, int64_t T, int32_t D,
                                  int32_t G, void* stream) {
  NOF_ARG(scan_types_ok(type, gate_type) && (reverse == 0 || reverse == 1));
  NOF_ARG(scan_sizes_ok(B, T, D, G) && gate_sb >= 0 && gate_st >= 0 && value_sb >= 0 && value_st >= 0);
  if (B == 0 || D == 0) return 0;
  NOF_ARG((gate && value) || T == 0);
  const int v = scan_vec(type, D, G);
  ScanArgs p = {};
  NOF_ARG(scan_plan(p, B, T, D, G, v, false));
  NOF_ARG(scan_aligned(value, value_sb, value_st, (int)learn_type_size(type), v) && scan_aligned(h, 0, 0, (int)learn_type_size(type), v));
  NOF_ARG(!p.per_channel || scan_aligned(gate, gate_sb, gate_st, (int)learn_type_size(gate_type), v));
  NOF_ARG(scan_aligned(state, 0, 0, 4, v) && scan_aligned(last, 0, 0, 4, v) && scan_aligned(marks, 0, 0, 4, v));
  NOF_ARG(p.segs == 1 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= scan_seg_bytes(p)));
  p.gate = gate; p.gate_sb = gate_sb; p.gate_st = gate_st;
  p.value = value; p.value_sb = value_sb; p.value_st = value_st;
  p.state = state; p.lengths = lengths; p.reverse = reverse;
  p.h = h; p.last = last; p.marks = marks;
  p.seg = (float*)workspace;
  LearnStream st = {(hipStream_t)stream, hipSuccess};
  const unsigned x = (unsigned)(B * p.tiles);
  if (p.segs > 1) SCAN_PICK(k_scan_segments, dim3(x, p.segs - 1), dim3(64 * p.waves), false);
  SCAN_PICK(k_scan_fwd, dim3(x, p.segs), dim3(64 * p.waves));
  LEARN_END(st);
  return 0;
}

extern "C" int nof_gated_scan_bwd(const void* gate, int64_t gate_sb, int64_t gate_st, int32_t gate_type, const void* value, int64_t value_sb,
                                  int64_t value_st, int32_t type, const void* dh, int64_t dh_sb, int64_t dh_st, const float* dlast,
                                  const float* marks, const int32_t* lengths, int32_t reverse, void* dgate, void* dvalue, float* dstate,
                                  void* workspace, int64_t workspace_bytes, int64_t B, int64_t T, int32_t D, int32_t G, void* stream) {
  NOF_ARG(scan_types_ok(type, gate_type) && (reverse == 0 || reverse == 1));
  NOF_ARG(scan_sizes_ok(B, T, D, G) && gate_sb >= 0 && gate_st >= 0 && value_sb >= 0 && value_st >= 0 && dh_sb >= 0 && dh_st >= 0);
  if (B == 0 || D == 0) return 0;
  NOF_ARG((gate && value && dh && marks && dgate && dvalue) || T == 0);
  const int v = scan_vec(type, D, G), size = (int)learn_type_size(type), gsize = (int)learn_type_size(gate_type);
  ScanArgs p = {};
  NOF_ARG(scan_plan(p, B, T, D, G, v, true));
  NOF_ARG(scan_aligned(value, value_sb, value_st, size, v) && scan_aligned(dh, dh_sb, dh_st, size, v) && scan_aligned(dvalue, 0, 0, size, v));
  NOF_ARG(!p.per_channel || (scan_aligned(gate, gate_sb, gate_st, gsize, v) && scan_aligned(dgate, 0, 0, gsize, v)));
  NOF_ARG(scan_aligned(dlast, 0, 0, 4, v) && scan_aligned(dstate, 0, 0, 4, v) && scan_aligned(marks, 0, 0, 4, v));
  const int64_t seg = scan_seg_bytes(p), gpart = scan_gpart_bytes(p);
  NOF_ARG(seg + gpart == 0 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= seg + gpart));
  p.gate = gate; p.gate_sb = gate_sb; p.gate_st = gate_st;
  p.value = value; p.value_sb = value_sb; p.value_st = value_st;
  p.dh = dh; p.dh_sb = dh_sb; p.dh_st = dh_st;
  p.dlast = dlast; p.marks = const_cast<float*>(marks); p.lengths = lengths; p.reverse = reverse;
  p.dgate = dgate; p.dvalue = dvalue; p.dstate = dstate;
  p.seg = (float*)workspace;
  p.gpart = (float*)((char*)workspace + seg);
  LearnStream st = {(hipStream_t)stream, hipSuccess};
  const unsigned x = (unsigned)(B * p.tiles);
  if (p.segs > 1) SCAN_PICK(k_scan_segments, dim3(x, p.segs - 1), dim3(64 * p.waves), true);
  SCAN_PICK(k_scan_bwd, dim3(x, p.segs), dim3(64 * p.waves));
  if (gpart > 0) {
    const int64_t n = B * T * G, blocks = nof_div_up(n, 256);
    const dim3 grid((unsigned)(blocks < 1 << 16 ? blocks : 1 << 16));
    if (gate_type == NOF_TYPE_F32) LEARN_LAUNCH(k_scan_gate_sum<float>, grid, dim3(256), 0, st, (const float*)p.gpart, (float*)dgate, n, p.tiles_per_span);
    else if (gate_type == NOF_TYPE_BF16) LEARN_LAUNCH(k_scan_gate_sum<__bf16>, grid, dim3(256), 0, st, (const float*)p.gpart, (__bf16*)dgate, n, p.tiles_per_span);
    else LEARN_LAUNCH(k_scan_gate_sum<_Float16>, grid, dim3(256), 0, st, (const float*)p.gpart, (_Float16*)dgate, n, p.tiles_per_span);
  }
  LEARN_END(st);
  return 0;
}

template <typename TG, typename T, int V>
static void scan_launch_step(const void* gate, int64_t gate_sb, const void* value, int64_t value_sb, const float* state, float* new_state,
                             void* h, int64_t B, int32_t D, int32_t G, LearnStream& st) {
  const int per_row = (int)nof_div_up(D, 256 * V);
  LEARN_LAUNCH((k_scan_step<TG, T, V>), dim3((unsigned)(B * per_row)), dim3(256), 0, st, (const TG*)gate, gate_sb, (const T*)value,
                     value_sb, state, new_state, (T*)h, (int)B, D, G, per_row);
}

extern "C" int nof_gated_scan_step(const void* gate, int64_t gate_sb, int32_t gate_type, const void* value, int64_t value_sb, int32_t type,
                                   const float* state, float* new_state, void* h, int64_t B, int32_t D, int32_t G, void* stream) {
  NOF_ARG(scan_types_ok(type, gate_type));
  NOF_ARG(scan_sizes_ok(B, 1, D, G) && gate_sb >= 0 && value_sb >= 0);
  if (B == 0 || D == 0) return 0;
  NOF_ARG(gate && value && state && new_state && h);
  const int v = scan_vec(type, D, G), size = (int)learn_type_size(type);
  NOF_ARG(B * nof_div_up(D, 256 * v) < (int64_t)1 << 24);             // (less than 2^32 threads)
  NOF_ARG(scan_aligned(value, value_sb, 0, size, v) && scan_aligned(h, 0, 0, size, v));
  NOF_ARG(G != D || scan_aligned(gate, gate_sb, 0, (int)learn_type_size(gate_type), v));
  NOF_ARG(scan_aligned(state, 0, 0, 4, v) && scan_aligned(new_state, 0, 0, 4, v));
  LearnStream st = {(hipStream_t)stream, hipSuccess};
#define SCAN_STEP(TG, T, V) scan_launch_step<TG, T, V>(gate, gate_sb, value, value_sb, state, new_state, h, B, D, G, st)
  if (type == NOF_TYPE_F32) SCAN_STEP(float, float, 1);
  else if (type == NOF_TYPE_BF16 && gate_type == type) { if (v == 2) SCAN_STEP(__bf16, __bf16, 2); else SCAN_STEP(__bf16, __bf16, 1); }
  else if (type == NOF_TYPE_BF16) { if (v == 2) SCAN_STEP(float, __bf16, 2); else SCAN_STEP(float, __bf16, 1); }
  else if (gate_type == type) { if (v == 2) SCAN_STEP(_Float16, _Float16, 2); else SCAN_STEP(_Float16, _Float16, 1); }
  else { if (v == 2) SCAN_STEP(float, _Float16, 2); else SCAN_STEP(float, _Float16, 1); }
#undef SCAN_STEP
  LEARN_END(st);
  return 0;
}
