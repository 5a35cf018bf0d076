// Gated linear recurrence along time with its backward pass and its single step (nof_gated_scan_*, include/nof_hip.h).
//
//   forward    h[t] = a[t] h[t-1] + x[t],  h[-1] = state               a: the gate, one per channel or one per group of P = D / G channels
//   backward   r[t] = dh[t] + a[t+1] r[t+1]  (the last position adds dlast)
//              dx[t] = r[t],  da[t] = sum over the group of r[t] h[t-1],  dstate = a[0] r[0]
//
// Bound by memory: the forward reads a, x and writes h once, the backward reads a, x, dh and writes da, dx.  Composition of two steps
// (a, b) then (a', b') is (a a', a' b + b'), so time is cut twice: a workgroup takes a CHUNK of positions at a time, each of its slots
// SCAN_U consecutive positions of one channel in registers; slots compose their (a, b) by shuffles within a wave and through LDS between
// waves, the state between chunks stays in registers, and the next chunk's loads are in flight meanwhile.  Where batch x channels give
// too few workgroups, time is also cut into segments: a first launch composes each segment, and every workgroup of the second folds
// the segments before its own.
//
// The backward needs h[t-1] in binary32, not as the output rounded it: the forward leaves the state in front of every chunk ("marks",
// 4 / chunk bytes per element), and the backward runs the chunk forward again from there.  Rounded states instead would cost the gate's
// gradient up to half a step of the value's type.
//
// Work is laid out as tiles of CT = 2^cs channels (times V per lane); 64 / CT positions side by side fill a wave where channels are few.
// A tile never spans two groups of a shared gate, so the gate's gradient is one sum over the tile's lanes; a group of several tiles adds
// them in a second launch, in order.
#include "nof_learn_dev.h"

#define SCAN_U 8
#define SCAN_MAXW 16                    // waves per workgroup at most

struct ScanArgs {
  const void* gate; const void* value; const void* dh;
  int64_t gate_sb, gate_st, value_sb, value_st, dh_sb, dh_st;        // elements between batches and positions
  const float* state;                   // [B, D] or NULL
  const int32_t* lengths;               // [B] or NULL
  void* h; float* last; float* marks;
  const float* dlast;
  void* dvalue; void* dgate; float* dstate; float* gpart;
  float* seg;                           // segment summaries
  int64_t T;
  int B, D, G, P;                       // P = channels per tile group (D where each channel has its gate)
  int cs, tiles_per_group, groups, tiles;
  int waves, chunk, n_chunks, segs, chunks_per_seg;
  int per_channel, reverse;
};

// position i of the recurrence (0 first) as a row of the tensors
__device__ __forceinline__ int64_t scan_row(const ScanArgs& p, int64_t n, int64_t i) { return p.reverse ? n - 1 - i : i; }

__device__ __forceinline__ int64_t scan_len(const ScanArgs& p, int b) {
  if (!p.lengths) return p.T;
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : n > p.T ? p.T : n;
}

// inclusive composition of the slots' (A, B) over the workgroup, in slot order (REV: from the last slot down).  On return (A, B) is the
// composition of all slots BEFORE this one (identity for the first), and (TA, TB) of all slots.  `sh` holds SCAN_MAXW * 64 * V pairs.
template <int V, bool REV>
__device__ __forceinline__ void scan_compose(float (&A)[V], float (&B)[V], float (&TA)[V], float (&TB)[V], int cs, int waves, float2* sh) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, ct = 1 << cs, sub = lane >> cs, nsub = 64 >> cs;
  const int at = REV ? nsub - 1 - sub : sub;
  for (int o = 1; o < nsub; o <<= 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float a = REV ? __shfl_down(A[v], o * ct) : __shfl_up(A[v], o * ct), b = REV ? __shfl_down(B[v], o * ct) : __shfl_up(B[v], o * ct);
      if (at >= o) { B[v] = A[v] * b + B[v]; A[v] *= a; }
    }
  }
  if (at == nsub - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) sh[(w * V + v) * ct + (lane & (ct - 1))] = make_float2(A[v], B[v]);
  }
  // exclusive within the wave
  if (nsub > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float a = REV ? __shfl_down(A[v], ct) : __shfl_up(A[v], ct), b = REV ? __shfl_down(B[v], ct) : __shfl_up(B[v], ct);
      A[v] = at > 0 ? a : 1.0f;
      B[v] = at > 0 ? b : 0.0f;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 1.0f; B[v] = 0.0f; }
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float pa = 1.0f, pb = 0.0f;
    TA[v] = 1.0f; TB[v] = 0.0f;
    for (int k = 0; k < waves; ++k) {
      const int q = REV ? waves - 1 - k : k;
      if (q == w) { pa = TA[v]; pb = TB[v]; }
      const float2 s = sh[(q * V + v) * ct + (lane & (ct - 1))];
      TB[v] = s.x * TB[v] + s.y;
      TA[v] *= s.x;
    }
    B[v] = A[v] * pb + B[v];
    A[v] *= pa;
  }
}

// SCAN_U positions from i0 on of one lane's channels; what lies outside [0, n) or the tile is the identity (gate 1, value 0)
template <typename T, int V>
__device__ __forceinline__ void scan_load(const T* __restrict__ x, int64_t st, const ScanArgs& p, int64_t n, int64_t i0, bool on, float fill, float (&f)[SCAN_U][V]) {
#pragma unroll
  for (int u = 0; u < SCAN_U; ++u) {
#pragma unroll
    for (int v = 0; v < V; ++v) f[u][v] = fill;
    if (on && i0 + u < n) lload<T, V>(x + scan_row(p, n, i0 + u) * st, f[u]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void scan_gate(const T* __restrict__ g, const ScanArgs& p, int64_t n, int64_t i0, bool on, float (&f)[SCAN_U][V]) {
  if (p.per_channel) {
    scan_load<T, V>(g, p.gate_st, p, n, i0, on, 1.0f, f);
  } else {
#pragma unroll
    for (int u = 0; u < SCAN_U; ++u) {
      float a = 1.0f;
      if (on && i0 + u < n) a = lf(g[scan_row(p, n, i0 + u) * p.gate_st]);
#pragma unroll
      for (int v = 0; v < V; ++v) f[u][v] = a;
    }
  }
}

struct ScanWhere { int b, ch, group, slot; bool on; int64_t n; };

template <int V>
__device__ __forceinline__ ScanWhere scan_where(const ScanArgs& p) {
  ScanWhere q;
  const int lane = threadIdx.x & 63, ct = 1 << p.cs;
  const int tile = blockIdx.x % p.tiles;
  q.b = blockIdx.x / p.tiles;
  q.group = tile / p.tiles_per_group;
  const int in_group = ((tile % p.tiles_per_group) * ct + (lane & (ct - 1))) * V;
  q.on = in_group < p.P;
  q.ch = q.group * p.P + (q.on ? in_group : 0);
  q.slot = (threadIdx.x >> 6) * (64 >> p.cs) + (lane >> p.cs);
  q.n = scan_len(p, q.b);
  return q;
}

// (A, B) of a segment, seg [B, tiles' channels D, segs] as two planes: what the forward's launch of segments folds
template <typename TG, typename T, int V, bool BACK>
__global__ __launch_bounds__(64 * SCAN_MAXW) void k_scan_segments(ScanArgs p) {
  __shared__ float2 sh[2][SCAN_MAXW * 64 * V];
  const ScanWhere q = scan_where<V>(p);
  const int seg = BACK ? blockIdx.y + 1 : blockIdx.y;               // nobody needs the forward's last or the backward's first
  const TG* g = (const TG*)p.gate + q.b * p.gate_sb + (p.per_channel ? q.ch : q.group);
  const T* x = BACK ? (const T*)p.dh + q.b * p.dh_sb + q.ch : (const T*)p.value + q.b * p.value_sb + q.ch;
  const int64_t st = BACK ? p.dh_st : p.value_st;
  const int64_t c0 = (int64_t)seg * p.chunks_per_seg, c1 = c0 + p.chunks_per_seg < p.n_chunks ? c0 + p.chunks_per_seg : p.n_chunks;
  float SA[V], SB[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { SA[v] = 1.0f; SB[v] = 0.0f; }
  float a[SCAN_U][V], x_[SCAN_U][V];
  int flip = 0;
  for (int64_t k = 0; k < c1 - c0; ++k, flip ^= 1) {
    const int64_t c = BACK ? c1 - 1 - k : c0 + k, i0 = c * p.chunk + (int64_t)q.slot * SCAN_U;
    if (c * p.chunk >= q.n) { if (BACK) continue; else break; }
    scan_gate<TG, V>(g, p, q.n, i0, q.on, a);
    scan_load<T, V>(x, st, p, q.n, i0, q.on, 0.0f, x_);
    float A[V], Bv[V], TA[V], TB[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 1.0f; Bv[v] = 0.0f; }
    if (BACK) {
      // carry into position t-1 is a[t] (dh[t] + carry): composition (a, a dh)
#pragma unroll
      for (int u = SCAN_U - 1; u >= 0; --u)
#pragma unroll
        for (int v = 0; v < V; ++v) { Bv[v] = a[u][v] * (x_[u][v] + Bv[v]); A[v] *= a[u][v]; }
    } else {
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) { Bv[v] = a[u][v] * Bv[v] + x_[u][v]; A[v] *= a[u][v]; }
    }
    scan_compose<V, BACK>(A, Bv, TA, TB, p.cs, p.waves, sh[flip]);
#pragma unroll
    for (int v = 0; v < V; ++v) { SB[v] = TA[v] * SB[v] + TB[v]; SA[v] *= TA[v]; }
  }
  if (q.slot == 0 && q.on) {
    float* out = p.seg + (((int64_t)seg * p.B + q.b) * 2) * p.D + q.ch;
    lstore<float, V>(out, SA);
    lstore<float, V>(out + p.D, SB);
  }
}

template <typename TG, typename T, int V>
__global__ __launch_bounds__(64 * SCAN_MAXW) void k_scan_fwd(ScanArgs p) {
  __shared__ float2 sh[2][SCAN_MAXW * 64 * V];
  const ScanWhere q = scan_where<V>(p);
  const TG* g = (const TG*)p.gate + q.b * p.gate_sb + (p.per_channel ? q.ch : q.group);
  const T* x = (const T*)p.value + q.b * p.value_sb + q.ch;
  T* h = p.h ? (T*)p.h + (int64_t)q.b * p.T * p.D + q.ch : nullptr;
  const int seg = blockIdx.y;
  const int64_t c0 = (int64_t)seg * p.chunks_per_seg, c1 = c0 + p.chunks_per_seg < p.n_chunks ? c0 + p.chunks_per_seg : p.n_chunks;
  float S[V];
#pragma unroll
  for (int v = 0; v < V; ++v) S[v] = 0.0f;
  if (p.state && q.on) lload<float, V>(p.state + (int64_t)q.b * p.D + q.ch, S);
  for (int k = 0; k < seg; ++k) {
    float A[V], Bv[V];
    const float* s = p.seg + (((int64_t)k * p.B + q.b) * 2) * p.D + q.ch;
    lload<float, V>(s, A);
    lload<float, V>(s + p.D, Bv);
#pragma unroll
    for (int v = 0; v < V; ++v) S[v] = A[v] * S[v] + Bv[v];
  }
  float a[SCAN_U][V], b[SCAN_U][V];
  scan_gate<TG, V>(g, p, q.n, c0 * p.chunk + (int64_t)q.slot * SCAN_U, q.on, a);
  scan_load<T, V>(x, p.value_st, p, q.n, c0 * p.chunk + (int64_t)q.slot * SCAN_U, q.on, 0.0f, b);
  int flip = 0;
  for (int64_t c = c0; c < c1; ++c, flip ^= 1) {
    const int64_t i0 = c * p.chunk + (int64_t)q.slot * SCAN_U;
    if (p.marks && q.slot == 0 && q.on) lstore<float, V>(p.marks + ((int64_t)q.b * p.n_chunks + c) * p.D + q.ch, S);
    if (c * p.chunk < q.n) {
      float A[V], Bv[V], TA[V], TB[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { A[v] = 1.0f; Bv[v] = 0.0f; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) { Bv[v] = a[u][v] * Bv[v] + b[u][v]; A[v] *= a[u][v]; }
      float a2[SCAN_U][V], b2[SCAN_U][V];
      const int64_t i1 = i0 + p.chunk;
      const bool more = c + 1 < c1;
      scan_gate<TG, V>(g, p, more ? q.n : 0, i1, q.on, a2);
      scan_load<T, V>(x, p.value_st, p, more ? q.n : 0, i1, q.on, 0.0f, b2);
      scan_compose<V, false>(A, Bv, TA, TB, p.cs, p.waves, sh[flip]);
      float s[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { s[v] = A[v] * S[v] + Bv[v]; S[v] = TA[v] * S[v] + TB[v]; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u) {
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = a[u][v] * s[v] + b[u][v];
        if (h && q.on && i0 + u < q.n) lstore<T, V>(h + scan_row(p, q.n, i0 + u) * p.D, s);
        if (p.last && q.on && i0 + u == q.n - 1) lstore<float, V>(p.last + (int64_t)q.b * p.D + q.ch, s);
      }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) { a[u][v] = a2[u][v]; b[u][v] = b2[u][v]; }
    }
    if (h && q.on) {                                                  // rows behind the sequence's end
      float z[V];
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = 0.0f;
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
        if (i0 + u >= q.n && i0 + u < p.T) lstore<T, V>(h + (i0 + u) * p.D, z);
    }
  }
  if (q.n == 0 && seg == 0 && q.slot == 0 && q.on && p.last) lstore<float, V>(p.last + (int64_t)q.b * p.D + q.ch, S);
}

// sum of f[u] over the 2^cs lanes of a tile, for all SCAN_U values: each exchange halves what is left to add, so 8 values over 64 lanes
// take 4 + 2 + 1 + 3 exchanges instead of 48.  Lane l ends with the sum of f[u], u = the top three bits of its index in the tile
// (for tiles of fewer lanes: of the value(s) that its bits name).
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

template <typename TG, typename T, int V>
__global__ __launch_bounds__(64 * SCAN_MAXW) void k_scan_bwd(ScanArgs p) {
  __shared__ float2 sh[2][SCAN_MAXW * 64 * V];
  const ScanWhere q = scan_where<V>(p);
  const int lane = threadIdx.x & 63, ct = 1 << p.cs, tile = blockIdx.x % p.tiles;
  const TG* g = (const TG*)p.gate + q.b * p.gate_sb + (p.per_channel ? q.ch : q.group);
  const T* x = (const T*)p.value + q.b * p.value_sb + q.ch;
  const T* dh = (const T*)p.dh + q.b * p.dh_sb + q.ch;
  T* dx = (T*)p.dvalue + (int64_t)q.b * p.T * p.D + q.ch;
  const int seg = blockIdx.y;
  const int64_t c0 = (int64_t)seg * p.chunks_per_seg, c1 = c0 + p.chunks_per_seg < p.n_chunks ? c0 + p.chunks_per_seg : p.n_chunks;
  float R[V];                                                       // what later positions hand to this one
#pragma unroll
  for (int v = 0; v < V; ++v) R[v] = 0.0f;
  if (p.dlast && q.on) lload<float, V>(p.dlast + (int64_t)q.b * p.D + q.ch, R);
  for (int k = p.segs - 1; k > seg; --k) {
    float A[V], Bv[V];
    const float* s = p.seg + (((int64_t)k * p.B + q.b) * 2) * p.D + q.ch;
    lload<float, V>(s, A);
    lload<float, V>(s + p.D, Bv);
#pragma unroll
    for (int v = 0; v < V; ++v) R[v] = A[v] * R[v] + Bv[v];
  }
  for (int64_t c = c1 - 1; c >= c0; --c) {
    const int64_t i0 = c * p.chunk + (int64_t)q.slot * SCAN_U;
    if (c * p.chunk < q.n) {
      float a[SCAN_U][V], b[SCAN_U][V], d[SCAN_U][V], A[V], Bv[V], A2[V], B2[V], TA[V], TB[V], m[V];
      scan_gate<TG, V>(g, p, q.n, i0, q.on, a);
      scan_load<T, V>(x, p.value_st, p, q.n, i0, q.on, 0.0f, b);
      scan_load<T, V>(dh, p.dh_st, p, q.n, i0, q.on, 0.0f, d);
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = 0.0f;
      if (q.on) lload<float, V>(p.marks + ((int64_t)q.b * p.n_chunks + c) * p.D + q.ch, m);
#pragma unroll
      for (int v = 0; v < V; ++v) { A[v] = 1.0f; Bv[v] = 0.0f; B2[v] = 0.0f; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) { Bv[v] = a[u][v] * Bv[v] + b[u][v]; A[v] *= a[u][v]; }
#pragma unroll
      for (int u = SCAN_U - 1; u >= 0; --u)
#pragma unroll
        for (int v = 0; v < V; ++v) B2[v] = a[u][v] * (d[u][v] + B2[v]);
#pragma unroll
      for (int v = 0; v < V; ++v) A2[v] = A[v];
      scan_compose<V, false>(A, Bv, TA, TB, p.cs, p.waves, sh[0]);
      float s[V], r[V];
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = A[v] * m[v] + Bv[v];
      scan_compose<V, true>(A2, B2, TA, TB, p.cs, p.waves, sh[1]);
#pragma unroll
      for (int v = 0; v < V; ++v) { r[v] = A2[v] * R[v] + B2[v]; R[v] = TA[v] * R[v] + TB[v]; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)                              // b: h before each position
#pragma unroll
        for (int v = 0; v < V; ++v) { const float x0 = b[u][v]; b[u][v] = s[v]; s[v] = a[u][v] * s[v] + x0; }
#pragma unroll
      for (int u = SCAN_U - 1; u >= 0; --u)                         // d: r; b: the gate's gradient
#pragma unroll
        for (int v = 0; v < V; ++v) { d[u][v] += r[v]; r[v] = a[u][v] * d[u][v]; b[u][v] *= d[u][v]; }
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
        if (q.on && i0 + u < q.n) {
          const int64_t row = scan_row(p, q.n, i0 + u);
          lstore<T, V>(dx + row * p.D, d[u]);
          if (p.per_channel) lstore<TG, V>((TG*)p.dgate + ((int64_t)q.b * p.T + row) * p.D + q.ch, b[u]);
        }
      if (!p.per_channel) {
        float f[SCAN_U];
#pragma unroll
        for (int u = 0; u < SCAN_U; ++u) {
          f[u] = 0.0f;
#pragma unroll
          for (int v = 0; v < V; ++v) f[u] += q.on ? b[u][v] : 0.0f;
        }
        scan_tile_sum(f, p.cs);
        // lane bits cs-1, cs-2, cs-3 chose between the upper and the lower half of what was left
        const int in = lane & (ct - 1);
        int left = SCAN_U, u0 = 0;
        for (int k = 0; k < 3 && k < p.cs; ++k) { left >>= 1; if (in >> (p.cs - 1 - k) & 1) u0 += left; }
        const int low = p.cs > 3 ? in & ((1 << (p.cs - 3)) - 1) : 0;
#pragma unroll
        for (int j = 0; j < SCAN_U; ++j)
          if (low == 0 && j < left && i0 + u0 + j < q.n) {
            const int64_t at = ((int64_t)q.b * p.T + scan_row(p, q.n, i0 + u0 + j)) * p.G + q.group;
            if (p.tiles_per_group == 1) ((TG*)p.dgate)[at] = lt<TG>(f[j]);
            else p.gpart[at * p.tiles_per_group + tile % p.tiles_per_group] = f[j];
          }
      }
      __syncthreads();                                              // sh is written again by the next chunk
    }
    if (q.on) {                                                       // rows behind the sequence's end have no gradient
      float z[V];
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = 0.0f;
#pragma unroll
      for (int u = 0; u < SCAN_U; ++u)
        if (i0 + u >= q.n && i0 + u < p.T) {
          lstore<T, V>(dx + (i0 + u) * p.D, z);
          const int64_t row = (int64_t)q.b * p.T + i0 + u;
          if (p.per_channel) lstore<TG, V>((TG*)p.dgate + row * p.D + q.ch, z);
          else if ((lane & (ct - 1)) == 0) {
            if (p.tiles_per_group == 1) ((TG*)p.dgate)[row * p.G + q.group] = lt<TG>(0.0f);
            else p.gpart[(row * p.G + q.group) * p.tiles_per_group + tile % p.tiles_per_group] = 0.0f;
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

template <typename TG, typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(const TG* __restrict__ gate, int64_t gate_st, const T* __restrict__ value, int64_t value_st,
                                                   const float* __restrict__ state, float* __restrict__ new_state, T* __restrict__ h, int B,
                                                   int D, int G, int blocks_per_row) {
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
static bool scan_plan(ScanArgs& p, int64_t B, int64_t T, int32_t D, int32_t G, int v) {
  p.T = T; p.B = (int)B; p.D = D; p.G = G;
  p.per_channel = G == D;
  p.groups = p.per_channel ? 1 : G;
  p.P = D / p.groups;
  const int nv = p.P / v;
  p.cs = learn_log2_up(nv < 64 ? nv : 64);
  p.tiles_per_group = (int)nof_div_up(nv, (int64_t)1 << p.cs);
  p.tiles = p.groups * p.tiles_per_group;
  const int64_t slots = nof_div_up(T, SCAN_U), per_wave = 64 >> p.cs;
  p.waves = 1;
  while (p.waves < SCAN_MAXW && p.waves * per_wave < slots) p.waves *= 2;
  p.chunk = (int)(p.waves * per_wave * SCAN_U);
  p.n_chunks = (int)nof_div_up(T, p.chunk);
  // segments: enough workgroups for two per compute unit, of two chunks at least
  const int64_t wgs = B * p.tiles, want = wgs > 0 ? nof_div_up(512, wgs) : 1, most = p.n_chunks / 2 > 1 ? p.n_chunks / 2 : 1;
  p.segs = (int)(want < most ? want : most);
  p.chunks_per_seg = (int)nof_div_up(p.n_chunks > 0 ? p.n_chunks : 1, p.segs);
  p.segs = (int)nof_div_up(p.n_chunks > 0 ? p.n_chunks : 1, p.chunks_per_seg);
  return wgs < (int64_t)1 << 31;
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

#define SCAN_PICK(KERNEL, GRID, BLOCK, ...)                                                                                            \
  do {                                                                                                                                \
    if (type == NOF_TYPE_F32) hipLaunchKernelGGL((KERNEL<float, float, 1 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                        \
    else if (type == NOF_TYPE_BF16 && gate_type == type) {                                                                            \
      if (v == 2) hipLaunchKernelGGL((KERNEL<__bf16, __bf16, 2 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                                  \
      else hipLaunchKernelGGL((KERNEL<__bf16, __bf16, 1 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                                         \
    } else if (type == NOF_TYPE_BF16) {                                                                                               \
      if (v == 2) hipLaunchKernelGGL((KERNEL<float, __bf16, 2 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                                   \
      else hipLaunchKernelGGL((KERNEL<float, __bf16, 1 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                                          \
    } else if (gate_type == type) {                                                                                                   \
      if (v == 2) hipLaunchKernelGGL((KERNEL<_Float16, _Float16, 2 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                              \
      else hipLaunchKernelGGL((KERNEL<_Float16, _Float16, 1 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                                     \
    } else {                                                                                                                          \
      if (v == 2) hipLaunchKernelGGL((KERNEL<float, _Float16, 2 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                                 \
      else hipLaunchKernelGGL((KERNEL<float, _Float16, 1 __VA_ARGS__>), GRID, BLOCK, 0, st, p);                                        \
    }                                                                                                                                 \
  } while (0)

static int64_t scan_seg_bytes(const ScanArgs& p) { return p.segs > 1 ? learn_align((int64_t)p.segs * p.B * 2 * p.D * 4) : 0; }
static int64_t scan_gpart_bytes(const ScanArgs& p) {
  return !p.per_channel && p.tiles_per_group > 1 ? learn_align((int64_t)p.B * p.T * p.G * p.tiles_per_group * 4) : 0;
}

extern "C" int64_t nof_gated_scan_marks_bytes(int64_t B, int64_t T, int32_t D, int32_t G, int32_t type) {
  if (!scan_sizes_ok(B, T, D, G) || !learn_type_ok(type)) return -1;
  if (B == 0 || D == 0) return 0;
  ScanArgs p = {};
  if (!scan_plan(p, B, T, D, G, scan_vec(type, D, G))) return -1;
  return (int64_t)p.B * p.n_chunks * p.D * 4;
}

extern "C" int64_t nof_gated_scan_workspace_bytes(int64_t B, int64_t T, int32_t D, int32_t G, int32_t type) {
  if (!scan_sizes_ok(B, T, D, G) || !learn_type_ok(type)) return -1;
  if (B == 0 || D == 0) return 0;
  ScanArgs p = {};
  if (!scan_plan(p, B, T, D, G, scan_vec(type, D, G))) return -1;
  return scan_seg_bytes(p) + scan_gpart_bytes(p);
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
  NOF_ARG(scan_plan(p, B, T, D, G, v));
  NOF_ARG(scan_aligned(value, value_sb, value_st, (int)learn_type_size(type), v) && scan_aligned(h, 0, 0, (int)learn_type_size(type), v));
  NOF_ARG(!p.per_channel || scan_aligned(gate, gate_sb, gate_st, (int)learn_type_size(gate_type), v));
  NOF_ARG(scan_aligned(state, 0, 0, 4, v) && scan_aligned(last, 0, 0, 4, v) && scan_aligned(marks, 0, 0, 4, v));
  NOF_ARG(p.segs == 1 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= scan_seg_bytes(p)));
  p.gate = gate; p.gate_sb = gate_sb; p.gate_st = gate_st;
  p.value = value; p.value_sb = value_sb; p.value_st = value_st;
  p.state = state; p.lengths = lengths; p.reverse = reverse;
  p.h = h; p.last = last; p.marks = marks;
  p.seg = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  const unsigned x = (unsigned)(B * p.tiles);
  if (p.segs > 1) SCAN_PICK(k_scan_segments, dim3(x, p.segs - 1), dim3(64 * p.waves), , false);
  SCAN_PICK(k_scan_fwd, dim3(x, p.segs), dim3(64 * p.waves));
  NOF_LAUNCH_OK();
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
  NOF_ARG(scan_plan(p, B, T, D, G, v));
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
  hipStream_t st = (hipStream_t)stream;
  const unsigned x = (unsigned)(B * p.tiles);
  if (p.segs > 1) SCAN_PICK(k_scan_segments, dim3(x, p.segs - 1), dim3(64 * p.waves), , true);
  SCAN_PICK(k_scan_bwd, dim3(x, p.segs), dim3(64 * p.waves));
  if (gpart > 0) {
    const int64_t n = B * T * G, blocks = nof_div_up(n, 256);
    const dim3 grid((unsigned)(blocks < 1 << 16 ? blocks : 1 << 16));
    if (gate_type == NOF_TYPE_F32) hipLaunchKernelGGL(k_scan_gate_sum<float>, grid, dim3(256), 0, st, (const float*)p.gpart, (float*)dgate, n, p.tiles_per_group);
    else if (gate_type == NOF_TYPE_BF16) hipLaunchKernelGGL(k_scan_gate_sum<__bf16>, grid, dim3(256), 0, st, (const float*)p.gpart, (__bf16*)dgate, n, p.tiles_per_group);
    else hipLaunchKernelGGL(k_scan_gate_sum<_Float16>, grid, dim3(256), 0, st, (const float*)p.gpart, (_Float16*)dgate, n, p.tiles_per_group);
  }
  NOF_LAUNCH_OK();
  return 0;
}

template <typename TG, typename T, int V>
static void scan_launch_step(const void* gate, int64_t gate_sb, const void* value, int64_t value_sb, const float* state, float* new_state,
                             void* h, int64_t B, int32_t D, int32_t G, hipStream_t st) {
  const int per_row = (int)nof_div_up(D, 256 * V);
  hipLaunchKernelGGL((k_scan_step<TG, T, V>), dim3((unsigned)(B * per_row)), dim3(256), 0, st, (const TG*)gate, gate_sb, (const T*)value,
                     value_sb, state, new_state, (T*)h, (int)B, D, G, per_row);
}

extern "C" int nof_gated_scan_step(const void* gate, int64_t gate_sb, int32_t gate_type, const void* value, int64_t value_sb, int32_t type,
                                   const float* state, float* new_state, void* h, int64_t B, int32_t D, int32_t G, void* stream) {
  NOF_ARG(scan_types_ok(type, gate_type));
  NOF_ARG(scan_sizes_ok(B, 1, D, G) && gate_sb >= 0 && value_sb >= 0);
  NOF_ARG(B * nof_div_up(D, 256) < (int64_t)1 << 31);
  if (B == 0 || D == 0) return 0;
  NOF_ARG(gate && value && state && new_state && h);
  const int v = scan_vec(type, D, G), size = (int)learn_type_size(type);
  NOF_ARG(scan_aligned(value, value_sb, 0, size, v) && scan_aligned(h, 0, 0, size, v));
  NOF_ARG(G != D || scan_aligned(gate, gate_sb, 0, (int)learn_type_size(gate_type), v));
  NOF_ARG(scan_aligned(state, 0, 0, 4, v) && scan_aligned(new_state, 0, 0, 4, v));
  hipStream_t st = (hipStream_t)stream;
#define SCAN_STEP(TG, T, V) scan_launch_step<TG, T, V>(gate, gate_sb, value, value_sb, state, new_state, h, B, D, G, st)
  if (type == NOF_TYPE_F32) SCAN_STEP(float, float, 1);
  else if (type == NOF_TYPE_BF16 && gate_type == type) { if (v == 2) SCAN_STEP(__bf16, __bf16, 2); else SCAN_STEP(__bf16, __bf16, 1); }
  else if (type == NOF_TYPE_BF16) { if (v == 2) SCAN_STEP(float, __bf16, 2); else SCAN_STEP(float, __bf16, 1); }
  else if (gate_type == type) { if (v == 2) SCAN_STEP(_Float16, _Float16, 2); else SCAN_STEP(_Float16, _Float16, 1); }
  else { if (v == 2) SCAN_STEP(float, _Float16, 2); else SCAN_STEP(float, _Float16, 1); }
#undef SCAN_STEP
  NOF_LAUNCH_OK();
  return 0;
}
