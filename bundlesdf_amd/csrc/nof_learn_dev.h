// What the learning operators' kernels share (nof_embed.hip, nof_scan.hip, nof_ortho.hip): the three element types of their tensors and
// vectors of them.  Arithmetic is binary32 throughout; a value is rounded to its tensor's type once, when it is stored (round to
// nearest even: off by at most half a step of that type).
#pragma once
#include "nof_common.h"

template <typename T, int V> struct alignas(sizeof(T) * V) LearnVec { T v[V]; };

template <typename T> __device__ __forceinline__ float lf(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T lt(float x) { return (T)x; }

template <typename T, int V> __device__ __forceinline__ void lload(const T* __restrict__ p, float (&f)[V]) {
  const LearnVec<T, V> x = *reinterpret_cast<const LearnVec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = lf(x.v[i]);
}
template <typename T, int V> __device__ __forceinline__ void lstore(T* __restrict__ p, const float (&f)[V]) {
  LearnVec<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.v[i] = lt<T>(f[i]);
  *reinterpret_cast<LearnVec<T, V>*>(p) = x;
}

static inline size_t learn_type_size(int32_t t) { return t == NOF_TYPE_F32 ? 4 : 2; }
static inline bool learn_type_ok(int32_t t) { return t == NOF_TYPE_F32 || t == NOF_TYPE_BF16 || t == NOF_TYPE_F16; }
static inline int learn_log2_up(int64_t n) { int b = 0; while (((int64_t)1 << b) < n) ++b; return b; }
static inline int64_t learn_align(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }

// A call's stream and the status of its launches.  A call of several ends with the first that fails, and says so: the runtime's last error is the
// last launch's, one that succeeds clears it, and what later launches read would not be there.
struct LearnStream { hipStream_t stream; hipError_t status; };
#define LEARN_LAUNCH(kernel, grid, block, lds, st, ...)                                     \
  do { if ((st).status == hipSuccess) {                                                     \
         hipLaunchKernelGGL(kernel, grid, block, lds, (st).stream, __VA_ARGS__);            \
         (st).status = hipGetLastError();                                                   \
       } } while (0)
#define LEARN_END(st)                                                                       \
  do { if ((st).status != hipSuccess) return nof_set_error((int)(st).status, "%s: %s", __func__, hipGetErrorString((st).status)); } while (0)
