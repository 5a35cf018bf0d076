// The orthogonalised update of a weight matrix by Newton-Schulz products on the matrix cores (nof_orthogonalize, include/nof_hip.h).
//
//   X = G / max(|G|_F, eps), transposed if it is taller than wide;  then `steps` times
//   A = X X^T        P = a I + b A + c A A        X <- P X
// so a singular value s of X goes to a s + b s^3 + c s^5 and the singular vectors stay.
//
// Bound by the matrix cores.  A and A A are symmetric: only the tiles on and above the diagonal are computed, each is stored twice.
// Operands are fp16 pairs hi + lo / 2048 of 4096 times the value: off by 2^-23 of the value, or by 2^-48 where that is more (hi is subnormal
// below 2^-26 and lo takes what it leaves; with lo as it is, it would be subnormal below 2^-15 already: rows of 1e-5 of the largest were off by
// 1e-4 so, and steps that lift them made them most of the result).  Products hi hi + (hi lo + lo hi) / 2048 accumulate in binary32, large and
// small apart: a product is off by 5 * 2^-24 at most where binary32 rounds it by 2^-24, at a third of the fp16 rate, which on this card is some
// three times the binary32 rate.  One fp16 product instead would be off by 2^-12 per step, which small singular values amplify by up to a^steps:
// 4 % for a matrix of rank 4 plus noise of 1e-4.  The norm is summed in 64 bits: an error of it is common to all values and the polynomial
// amplifies it.  Of at most 64 rows, A A is formed more exactly (ort_square).
//
// Matrices of at most 128 x 128 take one workgroup and one launch (k_ortho_small): X lives in accumulator registers, operands in LDS.
// Thin ones, of at most 128 on one side, take a launch a step (k_ortho_thin).  Larger ones are three launches a step over images of X, X^T,
// A, P in the workspace (four where the Gram product is cut, ort_cuts), every product C = L R^T with both operands' rows along the summed
// index, so X is stored in both orientations.
#include "nof_learn_dev.h"
#include "nof_mfma_dev.h"

#define ORT_SCALE 4096.0f               // operands hold 4096 times their value: |P| <= 15, |X| <= 2 stay below 65504
#define ORT_LESS 2048.0f                // and their small parts 2048 times theirs
#define ORT_SMALL 128
#define ORT_NORM_BLOCKS 512             // at most
#define ORT_MAX_STEPS 32

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void ort_split(float x, _Float16& hi, _Float16& lo) {
  hi = (_Float16)x;
  lo = (_Float16)((x - (float)hi) * ORT_LESS);
}

// a product is large + small / 2048
__device__ __forceinline__ void ort_mma3(f16x8 lh, f16x8 ll, f16x8 rh, f16x8 rl, f32x16& large, f32x16& small) {
  small = PrecF16::mma(lh, rl, small);
  small = PrecF16::mma(ll, rh, small);
  large = PrecF16::mma(lh, rh, large);
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

// Few rows leave little to average: an error of A A is one of all of X, and up to four steps amplify it.  So in matrices of at most 64 rows
// A A is more exact than pairs would give it: of 33 to 64 rows as products of three fp16 parts (33 bits), of at most 32 on the binary64 matrix
// cores.  Relative error against 64 bits, 24 random matrices each: 9 x 287 2.7e-7 (as pairs 8.0e-7, a binary32 computation 6.0e-7), 32 x 500
// 7.9e-7 (2.2e-6, 2.7e-6), 33 x 128 1.3e-6 (1.8e-6, 1.3e-6), 64 x 500 1.2e-6 (1.7e-6, 1.6e-6); from 65 rows on pairs are no worse than
// binary32 (128 x 1000: 5.7e-7 and 1.7e-6).  64 x 64 as three parts 21.7 us, as pairs 19.8; 16 x 16 on the binary64 cores 13.1, as pairs 14.4.
enum { ORT_PAIRS, ORT_THREE, ORT_WIDE };
__host__ __device__ constexpr int ort_square(int rt) { return rt == 1 ? ORT_WIDE : rt == 2 ? ORT_THREE : ORT_PAIRS; }
__host__ __device__ constexpr int ort_parts(int rt) { return ort_square(rt) == ORT_THREE ? 3 : 2; }        // planes of A's image
__device__ __forceinline__ void ort_split(float x, float less, _Float16& hi, _Float16& mid, _Float16& lo) {       // of x + less
  hi = (_Float16)x;
  const float rest = ((x - (float)hi) + less) * ORT_LESS;
  mid = (_Float16)rest;
  lo = (_Float16)((rest - (float)mid) * ORT_LESS);
}

// P = ca I + cb A + cc A A of at most 32 rows, 16 x 16 blocks on and above the diagonal shared by `waves`; A in rows of ORT_WIDE_ROW (whose
// loads touch every bank equally), P as pairs
#define ORT_WIDE_ROW 36
typedef double f64x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void ort_poly64(const double* a, int r, int w, int waves, int lane, float ca, float cb, float cc, _Float16* hi, _Float16* lo, int pitch) {
  const int blocks = (r + 15) / 16, l15 = lane & 15, l4 = lane >> 4;
  for (int t = w; t < blocks * (blocks + 1) / 2; t += waves) {
    const int bi = t == 2, bj = t > 0;
    const double *L = a + (16 * bi + l15) * ORT_WIDE_ROW + l4, *R = a + (16 * bj + l15) * ORT_WIDE_ROW + l4;
    f64x4 s = {};
    for (int k = 0; k < r; k += 16) {
#pragma unroll
      for (int q = 0; q < 16; q += 4) s = __builtin_amdgcn_mfma_f64_16x16x4f64(L[k + q], R[k + q], s, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * bi + 4 * e + l4, j = 16 * bj + l15;
      const double v = (i == j ? (double)ca : 0.0) + (double)cb * a[i * ORT_WIDE_ROW + j] + (double)cc * s[e];
      _Float16 h, l;
      ort_split((float)(v * ORT_SCALE), h, l);
      hi[j * pitch + i] = h;
      lo[j * pitch + i] = l;
      if (bi != bj) { hi[i * pitch + j] = h; lo[i * pitch + j] = l; }
    }
  }
}
// (P's image where it has no block meets zeros of X, and has to be a number there)
__device__ __forceinline__ void ort_clear(_Float16* image, int halves, int tid, int threads) {
  const f16x8 z = {};
  for (int q = tid * 8; q < halves; q += threads * 8) *(f16x8*)(image + q) = z;
}

// 32 x 32 tile of L R^T over 16 n columns, three parts each, planes apart
__device__ __forceinline__ void ort_mma6(const _Float16* L, const _Float16* R, int plane, int n, f32x16& large, f32x16& small) {
  f32x16 least = {};
#pragma unroll 2
  for (int q = 0; q < n; ++q) {
    const f16x8 lh = *(const f16x8*)(L + 16 * q), lm = *(const f16x8*)(L + plane + 16 * q), ll = *(const f16x8*)(L + 2 * plane + 16 * q);
    const f16x8 rh = *(const f16x8*)(R + 16 * q), rm = *(const f16x8*)(R + plane + 16 * q), rl = *(const f16x8*)(R + 2 * plane + 16 * q);
    least = PrecF16::mma(lh, rl, least);
    least = PrecF16::mma(ll, rh, least);
    least = PrecF16::mma(lm, rm, least);
    ort_mma3(lh, lm, rh, rm, large, small);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) small[e] += least[e] * (1.0f / ORT_LESS);
}

// ---- one workgroup a matrix -------------------------------------------------------------------------------------------------------
// One wave per 32 x 32 tile of X (r <= k after the turn; tiles rt x KT).  LDS: images of hi and lo, rows of 32 KT + 8 halves (the pad
// spreads a column's 16-byte reads over all banks; known at compile time, or sixteen row offsets per store stay live and spill).  The first
// pair holds X for the Gram product and X^T for the last one, the second A, then P: symmetric, so their tiles are stored turned, four
// halves at a time.  Bound by the chain of products, barriers and LDS round trips: 1.8 us a step for 16 x 16, 3.4 for 64 x 64,
// 8.2 for 128 x 128 (half of it the matrix cores); four waves of 2 x 2 tiles instead of sixteen of one read half as much LDS and take 1.4
// times as long.
struct OrtCoef { float c[3 * ORT_MAX_STEPS]; };

// RT: rows of tiles at most; `out` may be `g`
template <typename T, int KT, int RT>
__global__ __launch_bounds__(64 * KT * RT) void k_ortho_small(const T* g, T* out, int m, int n, int steps, OrtCoef coef, float eps) {
  extern __shared__ __attribute__((aligned(16))) char ort_lds[];
  constexpr int square = ort_square(RT);
  __shared__ double red[16], a64[square == ORT_WIDE ? 32 * ORT_WIDE_ROW : 1];
  const bool tall = m > n;
  const int r = tall ? n : m, k = tall ? m : n, rt = square != ORT_PAIRS ? RT : (r + 31) / 32;
  int tid = threadIdx.x;
  int hi = (tid >> 5) & 1, l31 = tid & 31, w = __builtin_amdgcn_readfirstlane(tid >> 6), ti = w / KT, tj = w % KT;      // rt * KT waves
  constexpr int px = 32 * KT + 8;
  _Float16* xh = (_Float16*)ort_lds;
  _Float16* xl = xh + 32 * KT * px;
  _Float16* ah = xl + 32 * KT * px;
  _Float16* al = ah + 32 * RT * px;
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
  if (square == ORT_WIDE) ort_clear(ah, 2 * 32 * RT * px, tid, 64 * KT * RT);
  const double f = ort_factor(ort_block_sum(s, red), eps);
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = (float)((double)x[e] * f);
  const bool gram = tj < rt;                                          // this wave also owns tile (ti, tj) of A and P
  for (int step = 0; step < steps; ++step) {
    asm volatile("" : "+v"(tid));                                     // (no instruction: lane places are formed in the step, not before the loop and spilled)
    hi = (tid >> 5) & 1; l31 = tid & 31; j = 32 * tj + l31;
    auto put = [&](_Float16* h, _Float16* l, const auto& y) {         // this wave's tile, turned: four i side by side to row j
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f16x4 h4, l4;
#pragma unroll
        for (int e = 0; e < 4; ++e) { _Float16 a, b; ort_split(y[4 * q + e], a, b); h4[e] = a; l4[e] = b; }
        const int at = j * px + 32 * ti + 8 * q + 4 * hi;
        *(f16x4*)(h + at) = h4;
        *(f16x4*)(l + at) = l4;
      }
    };
    const float ca = coef.c[3 * step], cb = coef.c[3 * step + 1], cc = coef.c[3 * step + 2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int at = (32 * ti + nloc(hi, e)) * px + j;
      ort_split(x[e], xh[at], xl[at]);
    }
    __syncthreads();
    const int li = (32 * ti + l31) * px + 8 * hi, ri = (32 * tj + l31) * px + 8 * hi, own = j * px + 32 * ti + 4 * hi;
    f32x16 acc = {}, sq = {}, acc2 = {}, sq2 = {};                    // (acc2, sq2: what the small parts add)
    if (gram) {
#pragma unroll 2
      for (int q = 0; q < 2 * KT; ++q) {
        const f16x8 lh = *(const f16x8*)(xh + li + 16 * q), ll = *(const f16x8*)(xl + li + 16 * q);
        const f16x8 rh = *(const f16x8*)(xh + ri + 16 * q), rl = *(const f16x8*)(xl + ri + 16 * q);
        ort_mma3(lh, ll, rh, rl, acc, acc2);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) { acc[e] *= 1.0f / ORT_SCALE; acc2[e] *= 1.0f / (ORT_SCALE * ORT_LESS); }         // 4096 A
      if (square == ORT_WIDE) {
#pragma unroll
        for (int e = 0; e < 16; ++e) a64[l31 * ORT_WIDE_ROW + nloc(hi, e)] = ((double)acc[e] + (double)acc2[e]) * (1.0 / ORT_SCALE);
      } else if (square == ORT_THREE) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f16x4 h4, m4, l4;
#pragma unroll
          for (int e = 0; e < 4; ++e) { _Float16 h, m, l; ort_split(acc[4 * q + e], acc2[4 * q + e], h, m, l); h4[e] = h; m4[e] = m; l4[e] = l; }
          *(f16x4*)(ah + own + 8 * q) = h4;
          *(f16x4*)(al + own + 8 * q) = m4;
          *(f16x4*)(al + 32 * RT * px + own + 8 * q) = l4;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] += acc2[e];
        put(ah, al, acc);
      }
    }
    __syncthreads();                                                  // X has been read, A is there
    put(xh, xl, x);                                                   // X^T over X
    if (square == ORT_WIDE) {
      ort_poly64(a64, r, w, KT, tid & 63, ca, cb, cc, ah, al, px);
    } else {
      if (square == ORT_THREE && gram) ort_mma6(ah + li, ah + ri, 32 * RT * px, 2 * rt, sq, sq2);
      else if (gram) {
#pragma unroll 2
        for (int q = 0; q < 2 * rt; ++q)
          ort_mma3(*(const f16x8*)(ah + li + 16 * q), *(const f16x8*)(al + li + 16 * q), *(const f16x8*)(ah + ri + 16 * q), *(const f16x8*)(al + ri + 16 * q), sq, sq2);
      }
      __syncthreads();                                                // A has been read
      if (gram) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float one = 32 * ti + nloc(hi, e) == j ? ca * ORT_SCALE : 0.0f, s2 = sq2[e] * (1.0f / (ORT_SCALE * ORT_LESS));
          if (square == ORT_THREE) acc[e] = (one + cb * acc[e] + cc * (sq[e] * (1.0f / ORT_SCALE))) + (cb * acc2[e] + cc * s2);
          else acc[e] = one + cb * acc[e] + cc * (sq[e] * (1.0f / ORT_SCALE) + s2);
        }
        put(ah, al, acc);
      }
    }
    __syncthreads();
    f32x16 y = {}, y2 = {};
#pragma unroll 2
    for (int q = 0; q < 2 * rt; ++q) {
      const int lo = (32 * ti + l31) * px + 16 * q + 8 * hi, ro = (32 * tj + l31) * px + 16 * q + 8 * hi;
      ort_mma3(*(const f16x8*)(ah + lo), *(const f16x8*)(al + lo), *(const f16x8*)(xh + ro), *(const f16x8*)(xl + ro), y, y2);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = (y[e] + y2[e] * (1.0f / ORT_LESS)) * (1.0f / ORT_SCALE);
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

// ---- thin matrices ----------------------------------------------------------------------------------------------------------------
// At most 128 on the shorter side, more on the longer: a launch a step instead of three.  A workgroup owns a stretch of X's columns, 128 at a
// time through LDS, and knows the Gram matrix as the sum of all workgroups' parts of it, which the launch before left behind: it forms A and
// P for itself, then X <- P X of its columns and the new part.  X stays in memory as the accumulators hold it.  Parts are added in the order
// of the workgroups.  64 x 1000 fp32: 52 us (as tiles of the larger matrices, whose Gram product is one tile's chain over the long side, twice that),
// 64 x 16384: 122 us (five times), 128 x 4096: 145 us (1.6 times).
struct OrtThin {
  const double* part; int n_part;
  float* x; const float* gram_in; float* gram_out;
  int m, n, r, k, tall, blocks, chunks; // chunks of 128 columns per workgroup
  float ca, cb, cc, eps;
};
#define ORT_FIRST 0                     // X from the update, its part of the Gram matrix
#define ORT_STEP 1
#define ORT_FINAL 2                     // a step to the result

// one wave's tile as memory holds it: sixteen values a lane, whole lines
__device__ __forceinline__ void ort_tile_load(const float* p, int lane, float (&x)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float4 v = *(const float4*)(p + q * 256 + lane * 4);
    x[4 * q] = v.x; x[4 * q + 1] = v.y; x[4 * q + 2] = v.z; x[4 * q + 3] = v.w;
  }
}
template <typename A> __device__ __forceinline__ void ort_tile_store(float* p, int lane, const A& x) {
#pragma unroll
  for (int q = 0; q < 4; ++q) *(float4*)(p + q * 256 + lane * 4) = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
}
// 32 x 32 tile of L R^T over 16 n columns; lo planes dl, dr halves behind
__device__ __forceinline__ void ort_tile_product(const _Float16* L, int dl, const _Float16* R, int dr, int n, f32x16& large, f32x16& small) {
#pragma unroll 2
  for (int q = 0; q < n; ++q)
    ort_mma3(*(const f16x8*)(L + 16 * q), *(const f16x8*)(L + dl + 16 * q), *(const f16x8*)(R + 16 * q), *(const f16x8*)(R + dr + 16 * q), large, small);
}

template <typename T, int RT, int MODE>
__global__ __launch_bounds__(256 * RT) void k_ortho_thin(const T* g, T* out, OrtThin p) {
  extern __shared__ __attribute__((aligned(16))) char ort_lds[];
  constexpr int square = ort_square(RT);
  __shared__ double red[4 * RT], a64[square == ORT_WIDE ? 32 * ORT_WIDE_ROW : 1];
  constexpr int PX = 136, PA = 32 * RT + 8, plane_x = 128 * PA > 32 * RT * PX ? 128 * PA : 32 * RT * PX, plane_a = 32 * RT * PA;
  _Float16* X = (_Float16*)ort_lds;                                   // X [32 RT][PX] or X^T [128][PA]
  _Float16* A = X + 2 * plane_x;                                      // A, then P, [32 RT][PA]
  const int b = blockIdx.x / p.blocks, block = blockIdx.x % p.blocks, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ti = w / 4, tj = w % 4;
  int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
  const bool gram = tj < RT;                                          // this wave also owns tile (ti, tj) of A and P
  const int si = p.tall ? 1 : p.n, sj = p.tall ? p.n : 1;
  g += (size_t)b * p.m * p.n;
  out += (size_t)b * p.m * p.n;
  auto put = [&](_Float16* image, int plane, int column, const auto& y) {       // this wave's tile, turned: four i side by side to row `column`
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f16x4 h4, l4;
#pragma unroll
      for (int e = 0; e < 4; ++e) { _Float16 h, l; ort_split(y[4 * q + e], h, l); h4[e] = h; l4[e] = l; }
      _Float16* at = image + column * PA + 32 * ti + 8 * q + 4 * hi;
      *(f16x4*)at = h4;
      *(f16x4*)(at + plane) = l4;
    }
  };
  double f = 0.0;
  if (MODE == ORT_FIRST) {
    double s = 0.0;
    for (int q = tid; q < p.n_part; q += 256 * RT) s += p.part[b * p.n_part + q];
    f = ort_factor(ort_block_sum(s, red), p.eps);
  } else if constexpr (square != ORT_PAIRS) {
    double a[4 * RT];                                                 // a tile of A by 4 / RT waves
#pragma unroll
    for (int e = 0; e < 4 * RT; ++e) a[e] = 0.0;
    const int tile = w * RT / 4, first = w * RT % 4;
    const float* in = p.gram_in + ((size_t)b * p.blocks * RT * RT + tile) * 1024 + first * 256 + lane * 4;
#pragma unroll 2
    for (int q = 0; q < p.blocks; q += 4) {                           // four in binary32: conversions to 64 bits are slow (64 x 16384: 119 us, 182 without)
#pragma unroll
      for (int c = 0; c < RT; ++c) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = q + u < p.blocks ? *(const float4*)(in + (size_t)(q + u) * RT * RT * 1024 + c * 256) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        a[4 * c] += (double)((v[0].x + v[1].x) + (v[2].x + v[3].x));
        a[4 * c + 1] += (double)((v[0].y + v[1].y) + (v[2].y + v[3].y));
        a[4 * c + 2] += (double)((v[0].z + v[1].z) + (v[2].z + v[3].z));
        a[4 * c + 3] += (double)((v[0].w + v[1].w) + (v[2].w + v[3].w));
      }
    }
    if constexpr (square == ORT_WIDE) {
      ort_clear(A, 2 * plane_a, tid, 256 * RT);
#pragma unroll
      for (int e = 0; e < 4; ++e) a64[l31 * ORT_WIDE_ROW + nloc(hi, 4 * w + e)] = a[e] * (1.0 / ORT_SCALE);
      __syncthreads();
      ort_poly64(a64, p.r, w, 4, lane, p.ca, p.cb, p.cc, A, A + plane_a, PA);
    } else {
#pragma unroll
      for (int c = 0; c < RT; ++c) {
        f16x4 h4, m4, l4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = (float)a[4 * c + e];
          _Float16 h, m, l;
          ort_split(x, (float)(a[4 * c + e] - (double)x), h, m, l);
          h4[e] = h; m4[e] = m; l4[e] = l;
        }
        _Float16* at = A + (tile % RT * 32 + l31) * PA + tile / RT * 32 + 8 * (first + c) + 4 * hi;
        *(f16x4*)at = h4;
        *(f16x4*)(at + plane_a) = m4;
        *(f16x4*)(at + 2 * plane_a) = l4;
      }
      __syncthreads();
      f32x16 sq = {}, sq2 = {}, pp;
      if (gram) {
        ort_mma6(A + (32 * ti + l31) * PA + 8 * hi, A + (32 * tj + l31) * PA + 8 * hi, plane_a, 2 * RT, sq, sq2);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const _Float16* at = A + (32 * tj + l31) * PA + 32 * ti + 8 * q + 4 * hi;
          const f16x4 h4 = *(const f16x4*)at, m4 = *(const f16x4*)(at + plane_a), l4 = *(const f16x4*)(at + 2 * plane_a);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float one = 32 * ti + nloc(hi, 4 * q + e) == 32 * tj + l31 ? p.ca * ORT_SCALE : 0.0f;
            pp[4 * q + e] = (one + p.cb * (float)h4[e] + p.cc * (sq[4 * q + e] * (1.0f / ORT_SCALE))) +
                          (p.cb * (((float)m4[e] + (float)l4[e] * (1.0f / ORT_LESS)) * (1.0f / ORT_LESS)) + p.cc * (sq2[4 * q + e] * (1.0f / (ORT_SCALE * ORT_LESS))));
          }
        }
      }
      __syncthreads();                                                  // A has been read
      if (gram) put(A, plane_a, 32 * tj + l31, pp);
    }
  } else {
    float a[16];
    f32x16 sq = {}, sq2 = {};
    if (gram) {
#pragma unroll
      for (int e = 0; e < 16; ++e) a[e] = 0.0f;
      const float* in = p.gram_in + ((size_t)b * p.blocks * RT * RT + ti * RT + tj) * 1024;
#pragma unroll 4
      for (int q = 0; q < p.blocks; ++q) {
        float y[16];
        ort_tile_load(in + (size_t)q * RT * RT * 1024, lane, y);
#pragma unroll
        for (int e = 0; e < 16; ++e) a[e] += y[e];
      }
      put(A, plane_a, 32 * tj + l31, a);
    }
    __syncthreads();
    if (gram) ort_tile_product(A + (32 * ti + l31) * PA + 8 * hi, plane_a, A + (32 * tj + l31) * PA + 8 * hi, plane_a, 2 * RT, sq, sq2);
    __syncthreads();
    if (gram) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        a[e] = (32 * ti + nloc(hi, e) == 32 * tj + l31 ? p.ca * ORT_SCALE : 0.0f) + p.cb * a[e] + p.cc * ((sq[e] + sq2[e] * (1.0f / ORT_LESS)) * (1.0f / ORT_SCALE));
      put(A, plane_a, 32 * tj + l31, a);
    }
  }
  f32x16 part = {}, less = {};
  for (int c = 0; c < p.chunks; ++c) {
    asm volatile("" : "+v"(tid));                                     // (no instruction: lane places are formed in the loop, not before it and spilled)
    lane = tid & 63; hi = lane >> 5; l31 = lane & 31;
    const int chunk = block * p.chunks + c, j = chunk * 128 + 32 * tj + l31;
    if (chunk * 128 >= p.k) break;
    float* at = p.x + (((size_t)(b * p.blocks + block) * p.chunks + c) * RT * 4 + w) * 1024;
    float x[16];
    if (MODE == ORT_FIRST) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = 32 * ti + nloc(hi, e);
        x[e] = i < p.r && j < p.k ? (float)((double)lf(g[(size_t)i * si + (size_t)j * sj]) * f) : 0.0f;
      }
    } else {
      ort_tile_load(at, lane, x);
      put(X, plane_x, 32 * tj + l31, x);
      __syncthreads();                                                // X^T is there (and P)
      f32x16 y = {}, y2 = {};
      ort_tile_product(A + (32 * ti + l31) * PA + 8 * hi, plane_a, X + (32 * tj + l31) * PA + 8 * hi, plane_x, 2 * RT, y, y2);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = (y[e] + y2[e] * (1.0f / ORT_LESS)) * (1.0f / ORT_SCALE);
    }
    if (MODE == ORT_FINAL) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = 32 * ti + nloc(hi, e);
        if (i < p.r && j < p.k) out[(size_t)i * si + (size_t)j * sj] = lt<T>(x[e] * (1.0f / ORT_SCALE));
      }
      __syncthreads();                                                // X^T has been read
    } else {
      ort_tile_store(at, lane, x);
      __syncthreads();
      _Float16* to = X + (32 * ti + 4 * hi) * PX + 32 * tj + l31;
#pragma unroll
      for (int e = 0; e < 16; ++e) ort_split(x[e], to[nloc(0, e) * PX], to[plane_x + nloc(0, e) * PX]);
      __syncthreads();
      if (gram) ort_tile_product(X + (32 * ti + l31) * PX + 8 * hi, plane_x, X + (32 * tj + l31) * PX + 8 * hi, plane_x, 8, part, less);
      __syncthreads();
    }
  }
  if (MODE != ORT_FINAL && gram) {
#pragma unroll
    for (int e = 0; e < 16; ++e) part[e] = (part[e] + less[e] * (1.0f / ORT_LESS)) * (1.0f / ORT_SCALE);         // 4096 of A
    ort_tile_store(p.gram_out + (((size_t)b * p.blocks + block) * RT * RT + ti * RT + tj) * 1024, lane, part);
  }
}

// ---- larger matrices --------------------------------------------------------------------------------------------------------------
// images of one matrix, in halves: X [rp][kp], X^T [kp][rp] twice (the last product reads one while it writes the other), A and P
// [rp][rp].  32 hi of a row lie next to their 32 lo, a cache line that one stage of a product reads whole (as planes, lines of which a
// stage read half, L2 held the products at 10 TB/s of useful and as much useless traffic).
// rp, kp: r and k up to whole tiles, zeros in between.
struct OrtArgs {
  _Float16* ws; size_t per;             // halves per matrix
  int r, k, rp, kp, m, n, tall;
  float ca, cb, cc;
  int cur;                              // which X^T holds X
  int tiles;                            // of a matrix in this launch
  int split; float* parts;              // the Gram product's long axis in `split` parts, joined by a launch of its own
};
__device__ __forceinline__ _Float16* ort_x(const OrtArgs& p, int b) { return p.ws + b * p.per; }
__device__ __forceinline__ _Float16* ort_xt(const OrtArgs& p, int b, int which) { return p.ws + b * p.per + (size_t)(1 + which) * 2 * p.rp * p.kp; }
__device__ __forceinline__ _Float16* ort_a(const OrtArgs& p, int b) { return p.ws + b * p.per + (size_t)6 * p.rp * p.kp; }
__device__ __forceinline__ _Float16* ort_p(const OrtArgs& p, int b) { return p.ws + b * p.per + (size_t)6 * p.rp * p.kp + (size_t)2 * p.rp * p.rp; }

// partial sums of squares, one per workgroup; V elements (16 bytes) per access where every matrix starts on a 16-byte border
template <typename T, int V>
__global__ __launch_bounds__(256) void k_ortho_norm(const T* __restrict__ g, int64_t count, double* __restrict__ part) {
  __shared__ double red[4];
  g += (size_t)blockIdx.y * count;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  const int64_t step = (int64_t)gridDim.x * 256 * V;
#pragma unroll 4
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < count; i += step) {
    float f[V];
    lload<T, V>(g + i, f);
#pragma unroll
    for (int q = 0; q < V; ++q) s[q & 3] += (double)f[q] * (double)f[q];
  }
  const double t = ort_block_sum((s[0] + s[1]) + (s[2] + s[3]), red);
  if (threadIdx.x == 0) part[blockIdx.y * gridDim.x + blockIdx.x] = t;
}

// where column `col` (of `ld`) of row `row` has its hi; its lo is 32 halves on
__device__ __forceinline__ size_t ort_at(int row, int col, int ld) { return (size_t)row * 2 * ld + (col >> 5) * 64 + (col & 31); }

// X and X^T of 4096 G / norm, tiles of 64 x 64 turned through LDS
template <typename T>
__global__ __launch_bounds__(256) void k_ortho_split(const T* __restrict__ g, const double* __restrict__ part, int n_part, OrtArgs p, float eps) {
  __shared__ double red[4];
  __shared__ float tile[64][65];
  const int b = blockIdx.z, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int rows = p.tall ? p.kp : p.rp, cols = p.tall ? p.rp : p.kp;  // of G's own orientation, padded
  const int y0 = blockIdx.y * 64, x0 = blockIdx.x * 64;
  g += (size_t)b * p.m * p.n;
  T v[16];                                                            // sixteen loads in flight, under the sum of the squares
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int gy = y0 + 4 * q + w, gx = x0 + lane;
    v[q] = gy < p.m && gx < p.n ? g[(size_t)gy * p.n + gx] : (T)0.0f;
  }
  double s = 0.0;
  for (int q = threadIdx.x; q < n_part; q += 256) s += part[b * n_part + q];
  const double f = ort_factor(ort_block_sum(s, red), eps);
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const bool in = y0 + 4 * q + w < p.m && x0 + lane < p.n;          // (padding stays zero where the norm is not finite)
    tile[4 * q + w][lane] = in ? (float)((double)lf(v[q]) * f) : 0.0f;
  }
  __syncthreads();
  _Float16* along = p.tall ? ort_xt(p, b, p.cur) : ort_x(p, b);        // [rows][cols]
  _Float16* turned = p.tall ? ort_x(p, b) : ort_xt(p, b, p.cur);       // [cols][rows]
#pragma unroll
  for (int q = 0; q < 4; ++q) {                                       // eight of a row of either: 16 bytes of hi, 16 of lo
    const int y = (q & 1) * 32 + threadIdx.x / 8, x = threadIdx.x % 8 * 8;
    f16x8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 hh, ll;
      ort_split(q < 2 ? tile[y][x + e] : tile[x + e][y], hh, ll);
      h[e] = hh;
      l[e] = ll;
    }
    _Float16* to = q < 2 ? along : turned;
    const int row = (q < 2 ? y0 : x0) + y, col = (q < 2 ? x0 : y0) + x, ld = q < 2 ? cols : rows;
    const size_t at = ort_at(row, col, ld);
    *(f16x8*)(to + at) = h;
    *(f16x8*)(to + at + 32) = l;
  }
}

#define ORT_GRAM 0
#define ORT_POLY 1
#define ORT_APPLY 2
#define ORT_LAST 3
#define ORT_JOIN 4                      // the Gram product's parts, added in order

// A stage is 64 halves of every row: 32 of the summed index as hi and lo.  16-byte piece c of row `row`
// sits at piece c ^ ort_swizzle(row): a fragment's reads (one piece of 32 consecutive rows) then touch every bank equally, for eight lanes
// of 128 bytes and for sixteen of 256
__device__ __forceinline__ int ort_swizzle(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// C = L R^T.  A workgroup is WM x WN waves of TI x TJ tiles of 32 x 32; a stage is 64 halves of every row, NS stages a ring in
// LDS that direct loads fill NS - 1 stages ahead, one barrier a stage.  Operands are pairs in every product, the last one of a 16-bit result
// too: of hi alone, bfloat16 results lay beyond the rounding's half step by 4.3e-4 of their norm (1024 x 1024 of rank 16), and so they would more
// with a larger first coefficient (P's diagonal is 4096 a, which fp16 steps by 8 and up).
// KG groups of such waves take the stages in turn, so that few tiles still give every SIMD several waves; their sums meet in LDS.
template <int WM, int WN, int TI, int TJ, int NS, int KG> struct OrtShape {
  static constexpr int wm = WM, wn = WN, ti = TI, tj = TJ, ns = NS, kg = KG, M = WM * TI * 32, N = WN * TJ * 32, group = WM * WN * 64, threads = group * KG;
  static constexpr int stage = 64 * (M + N), loads = stage / 8 / group;                            // halves of a stage; 16-byte pieces of it per thread
};
// counted wait for this thread's direct loads, its LDS reads done
template <int N> __device__ __forceinline__ void ort_wait() { __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070); }

// a wave's LDS writes are seen by its other lanes' reads behind this (LDS operations of a wave complete in order; this holds the compiler)
__device__ __forceinline__ void ort_wave_sync() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

template <int MODE, typename T, typename S>
__global__ __launch_bounds__(S::threads, S::threads / 256 * (S::ns * S::kg * S::stage <= 40960 ? 2 : 1)) void k_ortho_gemm(OrtArgs p, T* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) _Float16 lds[S::ns * S::kg * S::stage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, l31 = lane & 31;
  const int w = wave % (S::group / 64), kg = wave / (S::group / 64), tid = threadIdx.x % S::group;
  // Workgroups go round the eight XCDs: each takes a stretch of neighbouring tiles, whose operands its L2 then holds once
  const int total = gridDim.x, each = total / 8, more = total % 8, xcd = blockIdx.x % 8;
  int t = xcd * each + (xcd < more ? xcd : more) + blockIdx.x / 8, bi, bj;
  int slice = 0;                                                      // of the summed axis
  if (MODE == ORT_GRAM && p.split > 1) {                             
    const int whole = t / p.tiles;
    slice = whole % p.split;
    t -= (whole - whole / p.split) * p.tiles;                         // batch entry * tiles + tile
  }
  const int b = t / p.tiles;
  t -= b * p.tiles;
  const size_t part = ((size_t)b * p.tiles + t) * p.split * S::M * S::N;       // where the parts of this tile begin
  // within it, blocks of 8 x 8 tiles
  const int nt = p.rp / S::M;
  if (MODE == ORT_GRAM || MODE == ORT_POLY || MODE == ORT_JOIN) {     // tiles on and above the diagonal
    int bI = 0, bJ = 0;
    for (;;) {
      const int h = nt - 8 * bI < 8 ? nt - 8 * bI : 8, v = nt - 8 * bJ < 8 ? nt - 8 * bJ : 8, n = bI == bJ ? h * (h + 1) / 2 : h * v;
      if (t < n) {
        if (bI == bJ) {
          bi = 0;
          while (t >= h - bi) { t -= h - bi; ++bi; }
          bj = 8 * bJ + bi + t;
          bi += 8 * bI;
        } else {
          bi = 8 * bI + t % h;
          bj = 8 * bJ + t / h;
        }
        break;
      }
      t -= n;
      if (8 * ++bJ >= nt) bJ = ++bI;
    }
  } else {
    const int mt = p.kp / S::N, panel = t / (8 * mt), h = nt - 8 * panel < 8 ? nt - 8 * panel : 8;
    t -= panel * 8 * mt;
    bi = 8 * panel + t % h;
    bj = t / h;
  }
  const _Float16 *L, *R;
  int K;
  if (MODE == ORT_GRAM || MODE == ORT_JOIN) { L = R = ort_x(p, b); K = p.kp; }
  else if (MODE == ORT_POLY) { L = R = ort_a(p, b); K = p.rp; }
  else { L = ort_p(p, b); R = ort_xt(p, b, p.cur); K = p.rp; }
  constexpr int kstep = 32;
  int s0 = 0, s1 = MODE == ORT_JOIN ? 0 : K / kstep;                  // the stages of this part
  if (MODE == ORT_GRAM && p.split > 1) {
    const unsigned n = s1;                                            // (at most 512, in at most 64 parts)
    s0 = n * slice / p.split;
    s1 = n * (slice + 1) / p.split;
  }
  const size_t pitch = 2 * (size_t)K;
  // where this thread's pieces of a stage come from: L's rows, then R's
  const _Float16* src[S::loads];
#pragma unroll
  for (int q = 0; q < S::loads; ++q) {
    const bool left = q * S::group < 8 * S::M;                        // (a turn of the group lies within one of the two)
    const int piece = q * S::group + tid - (left ? 0 : 8 * S::M), row = piece / 8, c = (piece % 8) ^ ort_swizzle(row);
    src[q] = (left ? L + (size_t)(bi * S::M + row) * pitch : R + (size_t)(bj * S::N + row) * pitch) + (size_t)(s0 + kg) * 64 + c * 8;
  }
  auto load = [&](int slot) {
#pragma unroll
    for (int q = 0; q < S::loads; ++q) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src[q],
                                       (__attribute__((address_space(3))) void*)(lds + (slot * S::kg + kg) * S::stage + (q * S::group + w * 64) * 8), 16, 0, 0);
      src[q] += S::kg * 64;
    }
  };
  f32x16 acc[S::ti][S::tj] = {}, less[S::ti][S::tj] = {};
  const int wi = (w / S::wn) * S::ti * 32, wj = (w % S::wn) * S::tj * 32;
  const int n_stages = s1 - s0, rounds = (n_stages + S::kg - 1) / S::kg, stages = (n_stages - kg + S::kg - 1) / S::kg;      // this group's stages
#pragma unroll
  for (int q = 0; q < S::ns - 1; ++q)
    if (q < stages) load(q);
  int slot = 0, fill = S::ns - 1;
  for (int it = 0; it < rounds; ++it) {
    if (it + S::ns - 2 < stages) ort_wait<(S::ns - 2) * S::loads>(); else ort_wait<0>();      // stage `it` has landed (this wave's part)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();                                     // ... everybody's; and everybody has read the stage before
    asm volatile("" ::: "memory");
    if (it + S::ns - 1 < stages) load(fill);
    const _Float16* st = lds + (slot * S::kg + kg) * S::stage;
    if (it < stages) {
    constexpr int ahead = S::ti * S::tj > 4 ? 1 : kstep / 16;        // sixteens of the summed index whose fragments are read at once
#pragma unroll
    for (int k0 = 0; k0 < kstep / 16; k0 += ahead) {
      f16x8 lh[ahead][S::ti], ll[ahead][S::ti], rh[ahead][S::tj], rl[ahead][S::tj];
#pragma unroll
      for (int kk = 0; kk < ahead; ++kk) {
        const int c = 2 * (k0 + kk) + hi;
#pragma unroll
        for (int t = 0; t < S::ti; ++t) {
          const int row = wi + 32 * t + l31, o = row * 64, z = ort_swizzle(row);
          lh[kk][t] = *(const f16x8*)(st + o + (c ^ z) * 8);
          ll[kk][t] = *(const f16x8*)(st + o + ((c + 4) ^ z) * 8);
        }
#pragma unroll
        for (int t = 0; t < S::tj; ++t) {
          const int row = wj + 32 * t + l31, o = (S::M + row) * 64, z = ort_swizzle(row);
          rh[kk][t] = *(const f16x8*)(st + o + (c ^ z) * 8);
          rl[kk][t] = *(const f16x8*)(st + o + ((c + 4) ^ z) * 8);
        }
      }
#pragma unroll
      for (int kk = 0; kk < ahead; ++kk)
#pragma unroll
        for (int i = 0; i < S::ti; ++i)
#pragma unroll
          for (int j = 0; j < S::tj; ++j)
            ort_mma3(lh[kk][i], ll[kk][i], rh[kk][j], rl[kk][j], acc[i][j], less[i][j]);
    }
    }
    slot = slot + 1 == S::ns ? 0 : slot + 1;
    fill = fill + 1 == S::ns ? 0 : fill + 1;
  }
#pragma unroll
  for (int i = 0; i < S::ti; ++i)
#pragma unroll
    for (int j = 0; j < S::tj; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] += less[i][j][e] * (1.0f / ORT_LESS);
  // Results leave through LDS, a band of 32 rows of the wave's tile at a time, so that global stores are 16 bytes a lane and whole rows of
  // the tile: stored from the accumulators they were 2 bytes a lane, and 8 in the other orientation.
  constexpr int wmax = 32 * (S::ti > S::tj ? S::ti : S::tj) + 8;
  static_assert(S::ns * S::stage >= S::wm * S::wn * 32 * wmax && S::ns * S::stage >= S::wm * S::wn * 64 * 33, "the bands fit the ring");
  ort_wait<0>();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();                                       // the ring is free
  asm volatile("" ::: "memory");
  if (S::kg > 1) {                                                    // the first group adds the others' sums, in order, and goes on alone
    static_assert(S::ns * S::stage * S::kg >= 2 * (S::kg - 1) * S::M * S::N, "the sums fit the ring");
    float* sums = (float*)lds;
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < S::ti; ++i)
#pragma unroll
        for (int j = 0; j < S::tj; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) sums[(((kg - 1) * S::group / 64 + w) * S::ti * S::tj * 16 + (i * S::tj + j) * 16 + e) * 64 + lane] = acc[i][j][e];
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int g = 1; g < S::kg; ++g)
#pragma unroll
        for (int i = 0; i < S::ti; ++i)
#pragma unroll
          for (int j = 0; j < S::tj; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] += sums[(((g - 1) * S::group / 64 + w) * S::ti * S::tj * 16 + (i * S::tj + j) * 16 + e) * 64 + lane];
    }
    __syncthreads();
    if (kg > 0) return;
  }
  if constexpr (MODE == ORT_GRAM || MODE == ORT_JOIN) {
    float* mine = p.parts + part + (size_t)slice * S::M * S::N + w * S::ti * S::tj * 1024;
    if (MODE == ORT_GRAM && p.split > 1) {
#pragma unroll
      for (int i = 0; i < S::ti; ++i)
#pragma unroll
        for (int j = 0; j < S::tj; ++j) ort_tile_store(mine + (i * S::tj + j) * 1024, lane, acc[i][j]);
      return;
    }
    if (MODE == ORT_JOIN) {
#pragma unroll 4
      for (int q = 0; q < p.split; ++q) {
#pragma unroll
        for (int i = 0; i < S::ti; ++i)
#pragma unroll
          for (int j = 0; j < S::tj; ++j) {
            float x[16];
            ort_tile_load(mine + (size_t)q * S::M * S::N + (i * S::tj + j) * 1024, lane, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] += x[e];
          }
      }
    }
  }
  const int i0 = bi * S::M + wi, j0 = bj * S::N + wj;
  if (MODE == ORT_LAST) {
    T* o = out + (size_t)b * p.m * p.n;
    float* band = (float*)lds + w * 32 * 33;
#pragma unroll
    for (int i = 0; i < S::ti; ++i)
#pragma unroll
      for (int j = 0; j < S::tj; ++j) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = acc[i][j][e] * (1.0f / (ORT_SCALE * ORT_SCALE));
          if (p.tall) band[l31 * 33 + nloc(hi, e)] = v;
          else if (i0 + 32 * i + nloc(hi, e) < p.r && j0 + 32 * j + l31 < p.k) o[(size_t)(i0 + 32 * i + nloc(hi, e)) * p.n + j0 + 32 * j + l31] = lt<T>(v);
        }
        if (p.tall) {
          ort_wave_sync();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int y = 2 * e + hi;
            if (j0 + 32 * j + y < p.k && i0 + 32 * i + l31 < p.r) o[(size_t)(j0 + 32 * j + y) * p.n + i0 + 32 * i + l31] = lt<T>(band[y * 33 + l31]);
          }
          ort_wave_sync();
        }
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < S::ti; ++i)
#pragma unroll
    for (int j = 0; j < S::tj; ++j) {
      f32x16& v = acc[i][j];
      if (MODE == ORT_POLY) {                                         // A is symmetric: its column piece is read along a row
        const int col = j0 + 32 * j + l31, row0 = i0 + 32 * i + 4 * hi;
        const _Float16* a = ort_a(p, b) + ort_at(col, i0 + 32 * i, p.rp) + 4 * hi;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f16x4 h4 = *(const f16x4*)(a + 8 * q), l4 = *(const f16x4*)(a + 32 + 8 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[4 * q + e] = (row0 + 8 * q + e == col ? p.ca * ORT_SCALE : 0.0f) + p.cb * ((float)h4[e] + (float)l4[e] * (1.0f / ORT_LESS)) +
                           p.cc * (v[4 * q + e] * (1.0f / ORT_SCALE));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= 1.0f / ORT_SCALE;
      }
    }
  _Float16* c = MODE == ORT_GRAM || MODE == ORT_JOIN ? ort_a(p, b) : MODE == ORT_POLY ? ort_p(p, b) : ort_x(p, b);
  _Float16* ct = MODE == ORT_APPLY ? ort_xt(p, b, p.cur ^ 1) : c;
  const int ld = MODE == ORT_APPLY ? p.kp : p.rp;
  _Float16* band = lds + w * 32 * wmax;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (MODE == ORT_APPLY || bi != bj) {                              // as computed; a tile on the diagonal is its own mirror image
#pragma unroll
      for (int i = 0; i < S::ti; ++i) {
#pragma unroll
        for (int j = 0; j < S::tj; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            _Float16 h, l;
            ort_split(acc[i][j][e], h, l);
            band[nloc(hi, e) * wmax + 32 * j + l31] = half ? l : h;
          }
        ort_wave_sync();
#pragma unroll
        for (int q = 0; q < 2 * S::tj; ++q) {
          const int piece = q * 64 + lane, row = piece / (4 * S::tj), at = piece % (4 * S::tj) * 8;
          const size_t to = ort_at(i0 + 32 * i + row, j0 + at, ld) + 32 * half;
          *(f16x8*)(c + to) = *(const f16x8*)(band + row * wmax + at);
        }
        ort_wave_sync();
      }
    }
#pragma unroll
    for (int j = 0; j < S::tj; ++j) {                                 // and turned
#pragma unroll
      for (int i = 0; i < S::ti; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f16x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            _Float16 h, l;
            ort_split(acc[i][j][4 * q + e], h, l);
            x[e] = half ? l : h;
          }
          *(f16x4*)(band + l31 * wmax + 32 * i + 8 * q + 4 * hi) = x;
        }
      ort_wave_sync();
#pragma unroll
      for (int q = 0; q < 2 * S::ti; ++q) {
        const int piece = q * 64 + lane, row = piece / (4 * S::ti), at = piece % (4 * S::ti) * 8;
        const size_t to = ort_at(j0 + 32 * j + row, i0 + at, p.rp) + 32 * half;
        *(f16x8*)(ct + to) = *(const f16x8*)(band + row * wmax + at);
      }
      ort_wave_sync();
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
static bool ort_sizes_ok(int64_t batch, int64_t m, int64_t n) {
  return batch >= 0 && batch < 65536 && m >= 0 && m <= 16384 && n >= 0 && n <= 16384;
}
static bool ort_is_small(int64_t m, int64_t n) { return m <= ORT_SMALL && n <= ORT_SMALL; }
// The tile of a product: 128 x 128 where that occupies more than half of the 256 compute units, else 64 x 64; up to one tile a compute unit by
// eight waves of it.  Images are padded to whole tiles.  Five steps as 64 x 64 and as 128 x 128, by X's tiles of 128 x 128: 2048 x 1024 (128) 290
// and 314 us, 2500 x 1024 (160) 341 and 334, 3500 x 1024 (224) 396 and 370, 1920 x 2048 (240) 706 and 646; A and P of 2048 x 2048 (136)
// 836 and 790 of the whole.  As eight waves and as four: 1920 x 2048 646 and 661, 2048 x 2048 (256) 790 and 822.
typedef OrtShape<2, 2, 2, 2, 2, 1> OrtWide;
typedef OrtShape<2, 2, 2, 2, 2, 2> OrtWideDeep;                        // one workgroup per compute unit at most: all of LDS is its ring
typedef OrtShape<2, 2, 1, 1, 2, 2> OrtNarrow;
typedef OrtShape<2, 2, 1, 1, 2, 4> OrtNarrowDeep;
typedef OrtShape<2, 2, 1, 1, 2, 1> OrtSingle;                          // the join's
// The Gram product of few tiles over a long axis is cut along it: at most two workgroups a compute unit, and eight stages a part at least.
// Five steps of 200 x 4096: 251 us uncut, 147 cut; 600 x 2900: 273 and 221; 333 x 1001, 3 of them: 170 and 166.  Below 1024 the join costs
// more than the parts save (512 x 512: 142 and 149), and so it does with many tiles of a middling length (1024 x 1024: 210 and 219;
// 1024 x 2048: 288 and 284; 1024 x 4096: 415 and 389).  Parts of four stages gained nothing (200 x 4096: 153 and 171).
static int ort_cuts(int64_t batch, int64_t rp, int64_t kp) {
  const int64_t n = rp / 64, tiles = batch * n * (n + 1) / 2, most = kp / 256, want = 512 / tiles;
  if (kp < 1024 || want < 2 || kp * want < 6144) return 1;
  return (int)(want < most ? want : most);
}
static bool ort_wide(int64_t tiles_of_128) { return tiles_of_128 > 128; }
static int64_t ort_up(int64_t x, int64_t unit) { return nof_div_up(x, unit) * unit; }
static int64_t ort_unit(int64_t batch, int64_t r, int64_t k) { return ort_wide(batch * nof_div_up(r, 128) * nof_div_up(k, 128)) ? 128 : 64; }

// workgroups per thin matrix: what each reads of the others' parts grows with the square of the shorter side
static void ort_thin_plan(int64_t r, int64_t k, int& blocks, int& chunks) {
  const int rt = (int)nof_div_up(r, 32), all = (int)nof_div_up(k, 128), most = rt <= 2 ? 32 : 16;
  chunks = (int)nof_div_up(all, all < most ? all : most);
  blocks = (int)nof_div_up(all, chunks);
}
static bool ort_is_thin(int64_t m, int64_t n) { return (m <= ORT_SMALL) != (n <= ORT_SMALL); }

extern "C" int64_t nof_orthogonalize_workspace_bytes(int64_t batch, int64_t m, int64_t n) {
  if (!ort_sizes_ok(batch, m, n)) return -1;
  if (batch == 0 || m == 0 || n == 0 || ort_is_small(m, n)) return 0;
  if (ort_is_thin(m, n)) {
    int blocks, chunks;
    const int64_t rt = nof_div_up(m < n ? m : n, 32);
    ort_thin_plan(m < n ? m : n, m < n ? n : m, blocks, chunks);
    return learn_align(batch * ORT_NORM_BLOCKS * 8) + batch * blocks * (chunks * rt * 4 + 2 * rt * rt) * 4096;
  }
  const int64_t r = m < n ? m : n, k = m < n ? n : m, unit = ort_unit(batch, r, k), rp = ort_up(r, unit), kp = ort_up(k, unit);
  const int64_t split = ort_cuts(batch, rp, kp), side = rp / 64;
  return learn_align(batch * ORT_NORM_BLOCKS * 8) + batch * (6 * rp * kp + 4 * rp * rp) * 2 + (split > 1 ? batch * side * (side + 1) / 2 * split * 64 * 64 * 4 : 0);
}

template <typename T, int KT, int RT>
static void ort_launch_small(const void* g, void* out, int64_t batch, int64_t m, int64_t n, int32_t steps, const float* coef, float eps, LearnStream& st) {
  OrtCoef c = {};
  for (int i = 0; i < 3 * steps; ++i) c.c[i] = coef[i];
  const int rt = (int)nof_div_up(m < n ? m : n, 32);
  constexpr size_t lds = (size_t)2 * 32 * (2 * KT + ort_parts(RT) * RT) * (32 * KT + 8);      // 136 KiB for KT = RT = 4
  if (lds > 64 << 10) (void)hipFuncSetAttribute((const void*)&k_ortho_small<T, KT, RT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  LEARN_LAUNCH((k_ortho_small<T, KT, RT>), dim3((unsigned)batch), dim3(64 * rt * KT), lds, st, (const T*)g, (T*)out, (int)m, (int)n, steps, c, eps);
}

template <int MODE, typename S> static int64_t ort_tiles(const OrtArgs& p) {
  const int64_t ni = p.rp / S::M, nj = p.kp / S::N;
  return MODE == ORT_GRAM || MODE == ORT_POLY || MODE == ORT_JOIN ? ni * (ni + 1) / 2 : ni * nj;
}
template <int MODE, typename T, typename S>
static void ort_gemm(OrtArgs& p, T* out, int64_t batch, LearnStream& st) {
  p.tiles = (int)ort_tiles<MODE, S>(p);
  const int64_t parts = MODE == ORT_GRAM ? p.split : 1;
  LEARN_LAUNCH((k_ortho_gemm<MODE, T, S>), dim3((unsigned)(p.tiles * batch * parts)), dim3(S::threads), 0, st, p, out);
}
template <int MODE, typename T>
static void ort_product(OrtArgs& p, T* out, int64_t batch, LearnStream& st) {
  const int64_t wide = p.rp % 128 == 0 && p.kp % 128 == 0 ? batch * ort_tiles<MODE, OrtWide>(p) : 0;
  if constexpr (MODE == ORT_GRAM) {
    if (p.split > 1) {
      if (batch * ort_tiles<MODE, OrtNarrow>(p) * p.split > 256) ort_gemm<MODE, T, OrtNarrow>(p, out, batch, st);
      else ort_gemm<MODE, T, OrtNarrowDeep>(p, out, batch, st);
      return ort_gemm<ORT_JOIN, T, OrtSingle>(p, out, batch, st);
    }
  }
  if (wide > 256) ort_gemm<MODE, T, OrtWide>(p, out, batch, st);
  else if (ort_wide(wide)) ort_gemm<MODE, T, OrtWideDeep>(p, out, batch, st);
  else if (batch * ort_tiles<MODE, OrtNarrow>(p) > 256) ort_gemm<MODE, T, OrtNarrow>(p, out, batch, st);
  else ort_gemm<MODE, T, OrtNarrowDeep>(p, out, batch, st);
}

// the sums of squares, as many as it says
template <typename T>
static int ort_launch_norm(const void* g, double* part, int64_t batch, int64_t m, int64_t n, LearnStream& st) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool wide = ((uintptr_t)g & 15) == 0 && m * n % V == 0;
  const int64_t want = nof_div_up(m * n, 256 * 8 * (wide ? 4 : 1));
  const int n_part = (int)(want < ORT_NORM_BLOCKS ? want : ORT_NORM_BLOCKS);
  if (wide) LEARN_LAUNCH((k_ortho_norm<T, V>), dim3(n_part, (unsigned)batch), dim3(256), 0, st, (const T*)g, m * n, part);
  else LEARN_LAUNCH((k_ortho_norm<T, 1>), dim3(n_part, (unsigned)batch), dim3(256), 0, st, (const T*)g, m * n, part);
  return n_part;
}

template <typename T, int RT, int MODE>
static void ort_thin_step(const void* g, void* out, const OrtThin& p, int64_t batch, LearnStream& st) {
  constexpr int px = 128 * (32 * RT + 8) > 32 * RT * 136 ? 128 * (32 * RT + 8) : 32 * RT * 136;
  constexpr size_t lds = 2 * (size_t)(2 * px + ort_parts(RT) * 32 * RT * (32 * RT + 8));                              // 136 KiB for RT = 4
  if (lds > 64 << 10) (void)hipFuncSetAttribute((const void*)&k_ortho_thin<T, RT, MODE>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  LEARN_LAUNCH((k_ortho_thin<T, RT, MODE>), dim3((unsigned)(batch * p.blocks)), dim3(256 * RT), lds, st, (const T*)g, (T*)out, p);
}
template <typename T, int RT>
static void ort_launch_thin(const void* g, void* out, void* workspace, int64_t batch, int64_t m, int64_t n, int32_t steps, const float* coef, float eps,
                            LearnStream& st) {
  OrtThin p = {};
  p.m = (int)m; p.n = (int)n; p.tall = m > n; p.r = (int)(m < n ? m : n); p.k = (int)(m < n ? n : m); p.eps = eps;
  ort_thin_plan(p.r, p.k, p.blocks, p.chunks);
  double* part = (double*)workspace;
  p.part = part;
  p.n_part = ort_launch_norm<T>(g, part, batch, m, n, st);
  p.x = (float*)((char*)workspace + learn_align(batch * ORT_NORM_BLOCKS * 8));
  float* grams = p.x + (size_t)batch * p.blocks * p.chunks * RT * 4 * 1024;
  const size_t each = (size_t)batch * p.blocks * RT * RT * 1024;
  p.gram_out = grams;
  ort_thin_step<T, RT, ORT_FIRST>(g, out, p, batch, st);
  for (int s = 0; s < steps; ++s) {
    p.ca = coef[3 * s]; p.cb = coef[3 * s + 1]; p.cc = coef[3 * s + 2];
    p.gram_in = grams + (s & 1 ? each : 0);
    p.gram_out = grams + (s & 1 ? 0 : each);
    if (s + 1 < steps) ort_thin_step<T, RT, ORT_STEP>(g, out, p, batch, st);
    else ort_thin_step<T, RT, ORT_FINAL>(g, out, p, batch, st);
  }
}

template <typename T>
static void ort_launch(const void* g, void* out, void* workspace, int64_t batch, int64_t m, int64_t n, int32_t steps, const float* coef, float eps,
                       LearnStream& st) {
  const int64_t r = m < n ? m : n, k = m < n ? n : m;
  if (ort_is_small(m, n)) {
    const int kt = (int)nof_div_up(k, 32);
    auto small = r > 64 ? (kt == 3 ? ort_launch_small<T, 3, 3> : ort_launch_small<T, 4, 4>)
               : r > 32 ? (kt == 2 ? ort_launch_small<T, 2, 2> : kt == 3 ? ort_launch_small<T, 3, 2> : ort_launch_small<T, 4, 2>)
               : kt == 1 ? ort_launch_small<T, 1, 1> : kt == 2 ? ort_launch_small<T, 2, 1> : kt == 3 ? ort_launch_small<T, 3, 1> : ort_launch_small<T, 4, 1>;
    small(g, out, batch, m, n, steps, coef, eps, st);
    return;
  }
  if (ort_is_thin(m, n)) {
    const int rt = (int)nof_div_up(r, 32);
    if (rt == 1) ort_launch_thin<T, 1>(g, out, workspace, batch, m, n, steps, coef, eps, st);
    else if (rt == 2) ort_launch_thin<T, 2>(g, out, workspace, batch, m, n, steps, coef, eps, st);
    else if (rt == 3) ort_launch_thin<T, 3>(g, out, workspace, batch, m, n, steps, coef, eps, st);
    else ort_launch_thin<T, 4>(g, out, workspace, batch, m, n, steps, coef, eps, st);
    return;
  }
  const int64_t unit = ort_unit(batch, r, k);
  OrtArgs p = {};
  p.r = (int)r; p.k = (int)k; p.rp = (int)ort_up(r, unit); p.kp = (int)ort_up(k, unit);
  p.m = (int)m; p.n = (int)n; p.tall = m > n;
  p.per = (size_t)6 * p.rp * p.kp + (size_t)4 * p.rp * p.rp;
  double* part = (double*)workspace;
  p.ws = (_Float16*)((char*)workspace + learn_align(batch * ORT_NORM_BLOCKS * 8));
  p.split = ort_cuts(batch, p.rp, p.kp);
  p.parts = (float*)(p.ws + batch * p.per);
  const unsigned nb = (unsigned)batch;
  const int n_part = ort_launch_norm<T>(g, part, batch, m, n, st);
  LEARN_LAUNCH(k_ortho_split<T>, dim3((p.tall ? p.rp : p.kp) / 64, (p.tall ? p.kp : p.rp) / 64, nb), dim3(256), 0, st, (const T*)g,
                     (const double*)part, n_part, p, eps);
  for (int s = 0; s < steps; ++s, p.cur ^= 1) {
    p.ca = coef[3 * s]; p.cb = coef[3 * s + 1]; p.cc = coef[3 * s + 2];
    ort_product<ORT_GRAM, float>(p, nullptr, batch, st);
    ort_product<ORT_POLY, float>(p, nullptr, batch, st);
    if (s + 1 < steps) ort_product<ORT_APPLY, float>(p, nullptr, batch, st);
    else ort_product<ORT_LAST, T>(p, (T*)out, batch, st);
  }
}

// Where the singular values go: they start in [0, 1], and operands hold 4096 times |p| <= 15, |x| <= 2 without leaving fp16.  A step takes an
// interval to an interval, whose ends lie at the old ends or where the polynomial is level.  The first step (from 1 on) that leaves, or 0.
static int ort_leaves(const float* coef, int steps) {
  double lo = 0.0, hi = 1.0;
  for (int q = 0; q < steps; ++q) {
    const double a = coef[3 * q], b = coef[3 * q + 1], c = coef[3 * q + 2], was[2] = {lo, hi};
    double worst = 0.0;                                               // of |p|, at the squares' ends or where it is level
    bool first = true;
    auto at = [&](double s) {
      const double l = s * s, p = a + l * (b + l * c), y = s * p;
      if (!(fabs(p) <= worst)) worst = fabs(p);
      if (first || !(y >= lo)) lo = y;
      if (first || !(y <= hi)) hi = y;
      first = false;
    };
    auto inside = [&](double l) {                                     // s = sqrt(l) and -sqrt(l), where they lie in the interval
      if (!(l >= 0.0)) return;
      const double s = sqrt(l);
      if (s >= was[0] && s <= was[1]) at(s);
      if (-s >= was[0] && -s <= was[1]) at(-s);
    };
    at(was[0]);
    at(was[1]);
    inside(0.0);
    if (c != 0.0) inside(-b / (2.0 * c));
    // a + 3 b l + 5 c l^2 = 0
    const double d = 9.0 * b * b - 20.0 * a * c;
    if (d >= 0.0) {
      const double t = -0.5 * (3.0 * b + (b < 0.0 ? -sqrt(d) : sqrt(d)));
      if (c != 0.0) inside(t / (5.0 * c));
      if (t != 0.0) inside(a / t);
    }
    if (!(worst <= 15.0 && lo >= -2.0 && hi <= 2.0)) return q + 1;
  }
  return 0;
}

extern "C" int nof_orthogonalize(const void* update, void* out, int32_t type, int32_t steps, const float* h_coef, float eps, void* workspace,
                                 int64_t workspace_bytes, int64_t batch, int64_t m, int64_t n, void* stream) {
  NOF_ARG(learn_type_ok(type));
  NOF_ARG(ort_sizes_ok(batch, m, n));
  NOF_ARG(steps >= 1 && steps <= ORT_MAX_STEPS && h_coef && eps >= 0.0f && eps <= 3.0e38f);
  if (batch == 0 || m == 0 || n == 0) return 0;
  if (const int q = ort_leaves(h_coef, steps))
    return nof_set_error(-1, "%s: argument check failed: these coefficients take singular values out of [0, 2] (step %d)", __func__, q - 1);
  NOF_ARG(update && out);
  const int64_t need = nof_orthogonalize_workspace_bytes(batch, m, n);
  NOF_ARG(need == 0 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need));
  LearnStream st = {(hipStream_t)stream, hipSuccess};
  if (type == NOF_TYPE_F32) ort_launch<float>(update, out, workspace, batch, m, n, steps, h_coef, eps, st);
  else if (type == NOF_TYPE_BF16) ort_launch<__bf16>(update, out, workspace, batch, m, n, steps, h_coef, eps, st);
  else ort_launch<_Float16>(update, out, workspace, batch, m, n, steps, h_coef, eps, st);
  LEARN_END(st);
  return 0;
}
