/* Vocabulary shared by the language-model kernels (ga_embed.cuh,
 * ga_logprobs.cuh, ga_clipnorm.cuh): element conversion, leading dimensions,
 * aligned vectors over rows that start anywhere. */
#ifndef GA_LM_COMMON_CUH
#define GA_LM_COMMON_CUH
#include "cluda.h"
#include "ga_lm_ptx.cuh"

/* ---- element <-> arithmetic type ---- */
static __device__ __forceinline__ float ga__lm_get(ga_half v) { return ga_half2float(v); }
static __device__ __forceinline__ float ga__lm_get(ga_float v) { return v; }
static __device__ __forceinline__ double ga__lm_get(ga_double v) { return v; }
static __device__ __forceinline__ void ga__lm_put(ga_half *p, float v) { *p = ga_float2half(v); }
/* a double narrows to half through float: two roundings, each to nearest */
static __device__ __forceinline__ void ga__lm_put(ga_half *p, double v) { *p = ga_float2half((float)v); }
static __device__ __forceinline__ void ga__lm_put(ga_float *p, float v) { *p = v; }
static __device__ __forceinline__ void ga__lm_put(ga_float *p, double v) { *p = (float)v; }
static __device__ __forceinline__ void ga__lm_put(ga_double *p, float v) { *p = (double)v; }
static __device__ __forceinline__ void ga__lm_put(ga_double *p, double v) { *p = v; }

/* N elements moved by one access (N * sizeof(T) is 1, 2, 4, 8 or 16 bytes, or a multiple of 16) */
template <typename T, int N>
struct alignas((sizeof(T) * N) > 16 ? 16 : (sizeof(T) * N)) ga__lm_vec {
  T v[N];
};

#define GA_LM_MAXD 4

/* Byte offset of leading index i: the dimensions left after collapsing, last one fastest. */
template <int ND>
static __device__ __forceinline__ long long ga__lm_offset(unsigned long long i,
                                                          const unsigned long long *dims,
                                                          const long long *strs) {
  if (ND <= 1) return (long long)i * strs[0];
  long long p = 0;
  if (i <= 0xffffffffULL) { /* quotients of 32-bit numbers are several times cheaper */
    unsigned int r = (unsigned int)i;
#pragma unroll
    for (int d = ND - 1; d > 0; d--) {
      const unsigned int n = dims[d] > 0xffffffffULL ? 0xffffffffu : (unsigned int)dims[d];
      const unsigned int q = r / n;
      p += (long long)(r - q * n) * strs[d];
      r = q;
    }
    return p + (long long)r * strs[0];
  }
#pragma unroll
  for (int d = ND - 1; d > 0; d--) {
    const unsigned long long q = i / dims[d];
    p += (long long)(i - q * dims[d]) * strs[d];
    i = q;
  }
  return p + (long long)i * strs[0];
}
#endif
