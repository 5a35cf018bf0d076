// The orthogonalised update of a weight matrix by Newton-Schulz products on the matrix cores (nof_orthogonalize, include/nof_hip.h).
//
//   X = G / max(|G|_F, eps), transposed if it is taller than wide;  then `steps` times
//   A = X X^T        P = a I + b A + c A A        X <- P X
// so a singular value s of X goes to a s + b s^3 + c s^5 and the singular vectors stay.
//
// Bound by the matrix cores.  A and A A are symmetric: only the tiles on and above the diagonal are computed, each is stored twice.
// Operands are fp16 pairs hi + lo of 4096 times the value (rounding of lo: 2^-23 of the value, subnormals out of reach for what carries
// weight), products hi hi + hi lo + lo hi accumulate in binary32: as exact as a binary32 product at a third of the fp16 rate, which on
// this card is some three times the binary32 rate.  One fp16 product instead would be off by 2^-12 per step, which small singular values
// amplify by up to a^steps: 4 % for a matrix of rank 4 plus noise of 1e-4.  The norm is summed in 64 bits: an error of it is common to all
// values and the polynomial amplifies it.
//
// Matrices of at most 128 x 128 take one workgroup and one launch (k_ortho_small): X lives in accumulator registers, operands in LDS.
// Larger ones are three launches a step over images of X, X^T, A, P in the workspace, every product C = L R^T with both operands'
// rows along the summed index, so X is stored in both orientations.
#include "nof_learn_dev.h"
#include "nof_mfma_dev.h"

#define ORT_SCALE 4096.0f               // operands hold 4096 times their value: |P| <= 15, |X| <= 2 stay below 65504
#define ORT_TILE 128
#define ORT_KSTEP 32
#define ORT_SMALL 128
#define ORT_NORM_BLOCKS 64
#define ORT_MAX_STEPS 32

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void ort_split(float x, _Float16& hi, _Float16& lo) {
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

__device__ __forceinline__ f32x16 ort_mma3(f16x8 lh, f16x8 ll, f16x8 rh, f16x8 rl, f32x16 c) {
  c = PrecF16::mma(lh, rl, c);
  c = PrecF16::mma(ll, rh, c);
  return PrecF16::mma(lh, rh, c);
}

// sum over the workgroup's threads in a fixed order, given to all
__device__ __forceinline__ double ort_block_sum(double s, double* sh) {
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) t += sh[w];
  __syncthreads();
  return t;
}

// what takes a matrix of this sum of squares to 4096 X; a zero matrix stays zero also for eps = 0, and what is not a number stays so
__device__ __forceinline__ double ort_factor(double sumsq, float eps) {
  const double n = sqrt(sumsq), d = n < (double)eps ? (double)eps : n;
  return d == 0.0 ? 0.0 : (double)ORT_SCALE / d;
}

// ---- one workgroup a matrix -------------------------------------------------------------------------------------------------------
// One wave per 32 x 32 tile of X (r <= k after the turn; tiles rt x KT).  LDS: two pairs of images, rows of 32 KT + 8 halves (the pad
// spreads a column's 16-byte reads over all banks; known at compile time, or sixteen row offsets per store stay live and spill).  The first holds X for the Gram product and X^T for the last one, the second A, then P.
struct OrtCoef { float c[3 * ORT_MAX_STEPS]; };

template <typename T, int KT>
__global__ __launch_bounds__(64 * KT * KT) void k_ortho_small(const T* __restrict__ g, T* __restrict__ out, int m, int n, int steps, OrtCoef coef, float eps) {
  extern __shared__ __attribute__((aligned(16))) char ort_lds[];
  __shared__ double red[16];
  const bool tall = m > n;
  const int r = tall ? n : m, k = tall ? m : n, rt = (r + 31) / 32;
  int tid = threadIdx.x;
  int hi = (tid >> 5) & 1, l31 = tid & 31, w = __builtin_amdgcn_readfirstlane(tid >> 6), ti = w / KT, tj = w % KT;      // rt * KT waves
  constexpr int px = 32 * KT + 8, pa = px;
  _Float16* xh = (_Float16*)ort_lds;
  _Float16* xl = xh + 32 * KT * px;
  _Float16* ah = xl + 32 * KT * px;
  _Float16* al = ah + 32 * KT * pa;
  g += (size_t)blockIdx.x * m * n;
  out += (size_t)blockIdx.x * m * n;
  int j = 32 * tj + l31;
  const int si = tall ? 1 : n, sj = tall ? n : 1;
  float x[16];
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int i = 32 * ti + nloc(hi, e);
    x[e] = i < r && j < k ? lf(g[i * si + j * sj]) : 0.0f;
    s += (double)x[e] * (double)x[e];
  }
  const double f = ort_factor(ort_block_sum(s, red), eps);
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = (float)((double)x[e] * f);
  const bool gram = tj < rt;                                          // this wave also owns tile (ti, tj) of A and P
  for (int step = 0; step < steps; ++step) {
    asm volatile("" : "+v"(tid));                                     // (no instruction: lane places are formed in the step, not before the loop and spilled)
    hi = (tid >> 5) & 1; l31 = tid & 31; j = 32 * tj + l31;
    const float ca = coef.c[3 * step], cb = coef.c[3 * step + 1], cc = coef.c[3 * step + 2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int at = (32 * ti + nloc(hi, e)) * px + j;
      ort_split(x[e], xh[at], xl[at]);
    }
    __syncthreads();
    f32x16 acc = {}, sq = {};
    if (gram) {
      #pragma unroll 2
      for (int q = 0; q < 2 * KT; ++q) {
        const int lo = (32 * ti + l31) * px + 16 * q + 8 * hi, ro = (32 * tj + l31) * px + 16 * q + 8 * hi;
        acc = ort_mma3(*(const f16x8*)(xh + lo), *(const f16x8*)(xl + lo), *(const f16x8*)(xh + ro), *(const f16x8*)(xl + ro), acc);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {                                  // 4096 A
        acc[e] *= 1.0f / ORT_SCALE;
        const int at = (32 * ti + nloc(hi, e)) * pa + 32 * tj + l31;
        ort_split(acc[e], ah[at], al[at]);
      }
    }
    __syncthreads();                                                  // X has been read, A is there
#pragma unroll
    for (int q = 0; q < 4; ++q) {                                     // X^T over X: rows j, four i side by side
      f16x4 h4, l4;
#pragma unroll
      for (int e = 0; e < 4; ++e) { _Float16 a, b; ort_split(x[4 * q + e], a, b); h4[e] = a; l4[e] = b; }
      const int at = j * px + 32 * ti + 8 * q + 4 * hi;
      *(f16x4*)(xh + at) = h4;
      *(f16x4*)(xl + at) = l4;
    }
    if (gram) {
#pragma unroll 2
      for (int q = 0; q < 2 * rt; ++q) {
        const int lo = (32 * ti + l31) * pa + 16 * q + 8 * hi, ro = (32 * tj + l31) * pa + 16 * q + 8 * hi;
        sq = ort_mma3(*(const f16x8*)(ah + lo), *(const f16x8*)(al + lo), *(const f16x8*)(ah + ro), *(const f16x8*)(al + ro), sq);
      }
    }
    __syncthreads();                                                  // A has been read
    if (gram) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = 32 * ti + nloc(hi, e), at = i * pa + 32 * tj + l31;
        const float p = (i == 32 * tj + l31 ? ca * ORT_SCALE : 0.0f) + cb * acc[e] + cc * (sq[e] * (1.0f / ORT_SCALE));
        ort_split(p, ah[at], al[at]);
      }
    }
    __syncthreads();
    f32x16 y = {};
#pragma unroll 2
    for (int q = 0; q < 2 * rt; ++q) {
      const int lo = (32 * ti + l31) * pa + 16 * q + 8 * hi, ro = (32 * tj + l31) * px + 16 * q + 8 * hi;
      y = ort_mma3(*(const f16x8*)(ah + lo), *(const f16x8*)(al + lo), *(const f16x8*)(xh + ro), *(const f16x8*)(xl + ro), y);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = y[e] * (1.0f / ORT_SCALE);
    __syncthreads();
  }
  asm volatile("" : "+v"(tid));
  hi = (tid >> 5) & 1; j = 32 * tj + (tid & 31);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int i = 32 * ti + nloc(hi, e);
    if (i < r && j < k) out[i * si + j * sj] = lt<T>(x[e] * (1.0f / ORT_SCALE));
  }
}

// ---- larger matrices --------------------------------------------------------------------------------------------------------------
// images of one matrix, in halves: X [rp][kp], X^T [kp][rp] twice (the last product reads one while it writes the other), A and P
// [rp][rp]; each image is a hi plane followed by its lo plane.  rp, kp: r and k up to whole tiles, zeros in between.
struct OrtArgs {
  _Float16* ws; size_t per;             // halves per matrix
  int r, k, rp, kp, m, n, tall, nt;     // nt = rp / ORT_TILE
  float ca, cb, cc;
  int cur;                              // which X^T holds X
};
__device__ __forceinline__ _Float16* ort_x(const OrtArgs& p, int b) { return p.ws + b * p.per; }
__device__ __forceinline__ _Float16* ort_xt(const OrtArgs& p, int b, int which) { return p.ws + b * p.per + (size_t)(1 + which) * 2 * p.rp * p.kp; }
__device__ __forceinline__ _Float16* ort_a(const OrtArgs& p, int b) { return p.ws + b * p.per + (size_t)6 * p.rp * p.kp; }
__device__ __forceinline__ _Float16* ort_p(const OrtArgs& p, int b) { return p.ws + b * p.per + (size_t)6 * p.rp * p.kp + (size_t)2 * p.rp * p.rp; }

template <typename T>
__global__ __launch_bounds__(256) void k_ortho_norm(const T* __restrict__ g, int64_t count, double* __restrict__ part) {
  __shared__ double red[4];
  g += (size_t)blockIdx.y * count;
  double s = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)ORT_NORM_BLOCKS * 256) {
    const double x = (double)lf(g[i]);
    s += x * x;
  }
  s = ort_block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.y * ORT_NORM_BLOCKS + blockIdx.x] = s;
}

// X and X^T of 4096 G / norm, tiles of 64 x 64 turned through LDS
template <typename T>
__global__ __launch_bounds__(256) void k_ortho_split(const T* __restrict__ g, const double* __restrict__ part, OrtArgs p, float eps) {
  __shared__ float tile[64][65];
  const int b = blockIdx.z;
  double s = 0.0;
  for (int q = 0; q < ORT_NORM_BLOCKS; ++q) s += part[b * ORT_NORM_BLOCKS + q];
  const double f = ort_factor(s, eps);
  g += (size_t)b * p.m * p.n;
  const int rows = p.tall ? p.kp : p.rp, cols = p.tall ? p.rp : p.kp;  // of G's own orientation, padded
  const int y0 = blockIdx.y * 64, x0 = blockIdx.x * 64;
  _Float16* along = p.tall ? ort_xt(p, b, p.cur) : ort_x(p, b);        // [rows][cols]
  _Float16* turned = p.tall ? ort_x(p, b) : ort_xt(p, b, p.cur);       // [cols][rows]
  const size_t plane = (size_t)p.rp * p.kp;
  const int c = threadIdx.x & 63;
  for (int y = threadIdx.x >> 6; y < 64; y += 4) {
    const int gy = y0 + y, gx = x0 + c;
    const float v = gy < p.m && gx < p.n ? (float)((double)lf(g[(size_t)gy * p.n + gx]) * f) : 0.0f;
    tile[y][c] = v;
    _Float16 h, l;
    ort_split(v, h, l);
    along[(size_t)gy * cols + gx] = h;
    along[plane + (size_t)gy * cols + gx] = l;
  }
  __syncthreads();
  for (int y = threadIdx.x >> 6; y < 64; y += 4) {
    _Float16 h, l;
    ort_split(tile[c][y], h, l);
    turned[(size_t)(x0 + y) * rows + y0 + c] = h;
    turned[plane + (size_t)(x0 + y) * rows + y0 + c] = l;
  }
}

#define ORT_GRAM 0
#define ORT_POLY 1
#define ORT_APPLY 2
#define ORT_LAST 3

// 16-byte piece c of row `row` of a staged tile sits at piece c ^ ort_swizzle(row): a fragment's reads (one piece of 32 consecutive rows)
// then touch every bank equally
__device__ __forceinline__ int ort_swizzle(int row) { return ((row >> 1) & 3) ^ ((row >> 3) & 1); }

// C = L R^T in tiles of 128 x 128, four waves of 64 x 64, ORT_KSTEP of the summed index per stage, two stages in LDS filled by direct loads
template <int MODE, typename T>
__global__ __launch_bounds__(256, 2) void k_ortho_gemm(OrtArgs p, T* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) _Float16 lds[2][4][ORT_TILE * ORT_KSTEP];
  const int b = blockIdx.z, lane = threadIdx.x & 63, w = threadIdx.x >> 6, hi = lane >> 5, l31 = lane & 31;
  int bi, bj;
  if (MODE == ORT_GRAM || MODE == ORT_POLY) {                         // tiles on and above the diagonal
    int t = blockIdx.x;
    bi = 0;
    while (t >= p.nt - bi) { t -= p.nt - bi; ++bi; }
    bj = bi + t;
  } else {
    bi = blockIdx.x % p.nt;
    bj = blockIdx.x / p.nt;
  }
  const _Float16 *L, *R;
  size_t planeL, planeR;
  int K;
  if (MODE == ORT_GRAM) { L = R = ort_x(p, b); planeL = planeR = (size_t)p.rp * p.kp; K = p.kp; }
  else if (MODE == ORT_POLY) { L = R = ort_a(p, b); planeL = planeR = (size_t)p.rp * p.rp; K = p.rp; }
  else { L = ort_p(p, b); planeL = (size_t)p.rp * p.rp; R = ort_xt(p, b, p.cur); planeR = (size_t)p.rp * p.kp; K = p.rp; }
  L += (size_t)bi * ORT_TILE * K;
  R += (size_t)bj * ORT_TILE * K;
  auto load = [&](int stage, int k0) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {                                     // 2048 pieces of 16 bytes, 256 a turn
      const int plane = q >> 1, base = (q & 1) * 256 + w * 64, piece = base + lane, row = piece >> 2, c = (piece & 3) ^ ort_swizzle(row);
      const _Float16* src = (plane < 2 ? L + (plane & 1) * planeL : R + (plane & 1) * planeR) + (size_t)row * K + k0 + c * 8;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                       (__attribute__((address_space(3))) void*)(&lds[stage][plane][base * 8]), 16, 0, 0);
    }
  };
  f32x16 acc[2][2] = {};
  const int wi = (w >> 1) * 64, wj = (w & 1) * 64;
  load(0, 0);
  __builtin_amdgcn_s_waitcnt(0x0f70);                                 // vmcnt(0): the stage is in LDS
  __syncthreads();
  for (int k0 = 0, s = 0; k0 < K; k0 += ORT_KSTEP, s ^= 1) {
    if (k0 + ORT_KSTEP < K) load(s ^ 1, k0 + ORT_KSTEP);
#pragma unroll
    for (int kk = 0; kk < ORT_KSTEP / 16; ++kk) {
      f16x8 f[4][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int ra = wi + 32 * t + l31, rb = wj + 32 * t + l31, c = 2 * kk + hi;
        const int oa = ra * ORT_KSTEP + (c ^ ort_swizzle(ra)) * 8, ob = rb * ORT_KSTEP + (c ^ ort_swizzle(rb)) * 8;
        f[0][t] = *(const f16x8*)(&lds[s][0][oa]);
        f[1][t] = *(const f16x8*)(&lds[s][1][oa]);
        f[2][t] = *(const f16x8*)(&lds[s][2][ob]);
        f[3][t] = *(const f16x8*)(&lds[s][3][ob]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = ort_mma3(f[0][i], f[1][i], f[2][j], f[3][j], acc[i][j]);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
  }
  const size_t planeX = (size_t)p.rp * p.kp, planeA = (size_t)p.rp * p.rp;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i0 = bi * ORT_TILE + wi + 32 * i, col = bj * ORT_TILE + wj + 32 * j + l31;
      f32x16& v = acc[i][j];
      if (MODE == ORT_POLY) {                                         // A is symmetric: its column piece is read along a row
        const _Float16* a = ort_a(p, b) + (size_t)col * p.rp + i0 + 4 * hi;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f16x4 h4 = *(const f16x4*)(a + 8 * q), l4 = *(const f16x4*)(a + planeA + 8 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[4 * q + e] = (i0 + 8 * q + 4 * hi + e == col ? p.ca * ORT_SCALE : 0.0f) + p.cb * ((float)h4[e] + (float)l4[e]) +
                           p.cc * (v[4 * q + e] * (1.0f / ORT_SCALE));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= 1.0f / ORT_SCALE;
      }
      if (MODE == ORT_LAST) {
        T* o = out + (size_t)b * p.m * p.n;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int row = i0 + nloc(hi, e);
          if (row < p.r && col < p.k) o[p.tall ? (size_t)col * p.n + row : (size_t)row * p.n + col] = lt<T>(v[e] * (1.0f / ORT_SCALE));
        }
      } else {
        _Float16* c = MODE == ORT_GRAM ? ort_a(p, b) : MODE == ORT_POLY ? ort_p(p, b) : ort_x(p, b);
        _Float16* ct = MODE == ORT_APPLY ? ort_xt(p, b, p.cur ^ 1) : c;
        const size_t plane = MODE == ORT_APPLY ? planeX : planeA;
        const int ld = MODE == ORT_APPLY ? p.kp : p.rp;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f16x4 h4, l4;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            _Float16 h, l;
            ort_split(v[4 * q + e], h, l);
            h4[e] = h; l4[e] = l;
            if (MODE == ORT_APPLY || bi != bj) {
              const size_t at = (size_t)(i0 + 8 * q + 4 * hi + e) * ld + col;
              c[at] = h;
              c[plane + at] = l;
            }
          }
          const size_t at = (size_t)col * p.rp + i0 + 8 * q + 4 * hi;
          *(f16x4*)(ct + at) = h4;
          *(f16x4*)(ct + plane + at) = l4;
        }
      }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
static bool ort_sizes_ok(int64_t batch, int64_t m, int64_t n) {
  return batch >= 0 && batch < 65536 && m >= 0 && m <= 16384 && n >= 0 && n <= 16384;
}
static bool ort_is_small(int64_t m, int64_t n) { return m <= ORT_SMALL && n <= ORT_SMALL; }
static int64_t ort_up(int64_t x) { return nof_div_up(x, ORT_TILE) * ORT_TILE; }

extern "C" int64_t nof_orthogonalize_workspace_bytes(int64_t batch, int64_t m, int64_t n) {
  if (!ort_sizes_ok(batch, m, n)) return -1;
  if (batch == 0 || m == 0 || n == 0 || ort_is_small(m, n)) return 0;
  const int64_t rp = ort_up(m < n ? m : n), kp = ort_up(m < n ? n : m);
  return learn_align(batch * ORT_NORM_BLOCKS * 8) + batch * (6 * rp * kp + 4 * rp * rp) * 2;
}

template <typename T, int KT>
static void ort_launch_small(const void* g, void* out, int64_t batch, int64_t m, int64_t n, int32_t steps, const float* coef, float eps, hipStream_t st) {
  OrtCoef c = {};
  for (int i = 0; i < 3 * steps; ++i) c.c[i] = coef[i];
  const int rt = (int)nof_div_up(m < n ? m : n, 32);
  constexpr size_t lds = (size_t)4 * 2 * 32 * KT * (32 * KT + 8);    // 136 KiB for KT = 4
  if (lds > 64 << 10) (void)hipFuncSetAttribute((const void*)&k_ortho_small<T, KT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL((k_ortho_small<T, KT>), dim3((unsigned)batch), dim3(64 * rt * KT), lds, st, (const T*)g, (T*)out, (int)m, (int)n, steps, c, eps);
}

template <typename T>
static void ort_launch(const void* g, void* out, void* workspace, int64_t batch, int64_t m, int64_t n, int32_t steps, const float* coef, float eps,
                       hipStream_t st) {
  const int64_t r = m < n ? m : n, k = m < n ? n : m;
  if (ort_is_small(m, n)) {
    const int kt = (int)nof_div_up(k, 32);
    if (kt == 1) ort_launch_small<T, 1>(g, out, batch, m, n, steps, coef, eps, st);
    else if (kt == 2) ort_launch_small<T, 2>(g, out, batch, m, n, steps, coef, eps, st);
    else if (kt == 3) ort_launch_small<T, 3>(g, out, batch, m, n, steps, coef, eps, st);
    else ort_launch_small<T, 4>(g, out, batch, m, n, steps, coef, eps, st);
    return;
  }
  OrtArgs p = {};
  p.r = (int)r; p.k = (int)k; p.rp = (int)ort_up(r); p.kp = (int)ort_up(k);
  p.m = (int)m; p.n = (int)n; p.tall = m > n;
  p.nt = p.rp / ORT_TILE;
  p.per = (size_t)6 * p.rp * p.kp + (size_t)4 * p.rp * p.rp;
  double* part = (double*)workspace;
  p.ws = (_Float16*)((char*)workspace + learn_align(batch * ORT_NORM_BLOCKS * 8));
  const unsigned nb = (unsigned)batch, sym = (unsigned)(p.nt * (p.nt + 1) / 2), full = (unsigned)(p.nt * (p.kp / ORT_TILE));
  hipLaunchKernelGGL(k_ortho_norm<T>, dim3(ORT_NORM_BLOCKS, nb), dim3(256), 0, st, (const T*)g, m * n, part);
  hipLaunchKernelGGL(k_ortho_split<T>, dim3((p.tall ? p.rp : p.kp) / 64, (p.tall ? p.kp : p.rp) / 64, nb), dim3(256), 0, st, (const T*)g,
                     (const double*)part, p, eps);
  for (int s = 0; s < steps; ++s, p.cur ^= 1) {
    p.ca = coef[3 * s]; p.cb = coef[3 * s + 1]; p.cc = coef[3 * s + 2];
    hipLaunchKernelGGL((k_ortho_gemm<ORT_GRAM, float>), dim3(sym, 1, nb), dim3(256), 0, st, p, (float*)nullptr);
    hipLaunchKernelGGL((k_ortho_gemm<ORT_POLY, float>), dim3(sym, 1, nb), dim3(256), 0, st, p, (float*)nullptr);
    if (s + 1 < steps) hipLaunchKernelGGL((k_ortho_gemm<ORT_APPLY, float>), dim3(full, 1, nb), dim3(256), 0, st, p, (float*)nullptr);
    else hipLaunchKernelGGL((k_ortho_gemm<ORT_LAST, T>), dim3(full, 1, nb), dim3(256), 0, st, p, (T*)out);
  }
}

extern "C" int nof_orthogonalize(const void* update, void* out, int32_t type, int32_t steps, const float* h_coef, float eps, void* workspace,
                                 int64_t workspace_bytes, int64_t batch, int64_t m, int64_t n, void* stream) {
  NOF_ARG(learn_type_ok(type));
  NOF_ARG(ort_sizes_ok(batch, m, n));
  NOF_ARG(steps >= 1 && steps <= ORT_MAX_STEPS && h_coef && eps >= 0.0f && eps <= 3.0e38f);
  if (batch == 0 || m == 0 || n == 0) return 0;
  // where the singular values go: they start in [0, 1], and operands hold 4096 times |p| <= 15, |x| <= 2 without leaving fp16
  {
    double s[129];
    for (int i = 0; i <= 128; ++i) s[i] = i / 128.0;
    for (int q = 0; q < steps; ++q)
      for (int i = 0; i <= 128; ++i) {
        const double l = s[i] * s[i], f = (double)h_coef[3 * q] + l * ((double)h_coef[3 * q + 1] + l * (double)h_coef[3 * q + 2]);
        s[i] *= f;
        if (!(fabs(f) <= 15.0 && fabs(s[i]) <= 2.0))
          return nof_set_error(-1, "%s: argument check failed: these coefficients take singular values out of [0, 2] (step %d)", __func__, q);
      }
  }
  NOF_ARG(update && out);
  const int64_t need = nof_orthogonalize_workspace_bytes(batch, m, n);
  NOF_ARG(need == 0 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need));
  hipStream_t st = (hipStream_t)stream;
  if (type == NOF_TYPE_F32) ort_launch<float>(update, out, workspace, batch, m, n, steps, h_coef, eps, st);
  else if (type == NOF_TYPE_BF16) ort_launch<__bf16>(update, out, workspace, batch, m, n, steps, h_coef, eps, st);
  else ort_launch<_Float16>(update, out, workspace, batch, m, n, steps, h_coef, eps, st);
  NOF_LAUNCH_OK();
  return 0;
}
