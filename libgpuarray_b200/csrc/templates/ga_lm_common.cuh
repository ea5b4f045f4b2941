/* Vocabulary shared by the language-model kernels (ga_embed.cuh,
 * ga_logprobs.cuh, ga_clipnorm.cuh): element conversion, leading dimensions,
 * aligned vectors over rows that start anywhere. */
#ifndef GA_LM_COMMON_CUH
#define GA_LM_COMMON_CUH
#include "cluda.h"
#include "ga_lm_ptx.cuh"

/* ---- N elements of type T moved by one access, and as arithmetic type F ----
 *
 * They travel as 32-bit words, up to 8 of them: vectors declared as arrays of 2-byte elements
 * are taken apart into as many loads or byte moves. */
template <int BYTES> /* 4 to 32, a power of two */
struct alignas(BYTES) ga__lm_raw {
  unsigned int w[BYTES / 4];
};
template <>
struct alignas(2) ga__lm_raw<2> {
  unsigned short w[1];
};
template <typename T, int N>
using ga__lm_vec = ga__lm_raw<(int)sizeof(T) * N>;

template <typename R>
static __device__ __forceinline__ R ga__lm_load(const char *p) {
  if constexpr (sizeof(R) == 32) {
    R q;
    ga__ld32(q.w, p);
    return q;
  } else {
    return *reinterpret_cast<const R *>(p);
  }
}
template <typename R>
static __device__ __forceinline__ void ga__lm_store(char *p, const R &q) {
  if constexpr (sizeof(R) == 32) ga__st32(p, q.w);
  else *reinterpret_cast<R *>(p) = q;
}

template <typename T>
struct ga__lm_type;
template <>
struct ga__lm_type<ga_half> {
  template <int N, typename F>
  static __device__ __forceinline__ void get(F x[N], const ga__lm_raw<2 * N> &q) {
    if constexpr (N == 1) {
      ga_half h;
      h.data = (ga_ushort)q.w[0];
      x[0] = (F)ga_half2float(h);
    } else {
#pragma unroll
      for (int j = 0; j < N / 2; j++) {
        float a, b;
        ga__unpack_h2(q.w[j], a, b);
        x[2 * j] = (F)a;
        x[2 * j + 1] = (F)b;
      }
    }
  }
  /* one rounding: a double does not go by way of float */
  template <int N, typename F>
  static __device__ __forceinline__ void put(ga__lm_raw<2 * N> &q, const F x[N]) {
    if constexpr (sizeof(F) == 8) {
#pragma unroll
      for (int j = 0; j < (N + 1) / 2; j++) {
        q.w[j] = ga__half_bits((double)x[2 * j]);
        if constexpr (N > 1) q.w[j] |= (unsigned int)ga__half_bits((double)x[2 * j + 1]) << 16;
      }
    } else if constexpr (N == 1) {
      q.w[0] = ga_float2half((float)x[0]).data;
    } else {
#pragma unroll
      for (int j = 0; j < N / 2; j++) q.w[j] = ga__pack_h2((float)x[2 * j], (float)x[2 * j + 1]);
    }
  }
};
template <>
struct ga__lm_type<ga_float> {
  template <int N, typename F>
  static __device__ __forceinline__ void get(F x[N], const ga__lm_raw<4 * N> &q) {
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = (F)__uint_as_float(q.w[j]);
  }
  template <int N, typename F>
  static __device__ __forceinline__ void put(ga__lm_raw<4 * N> &q, const F x[N]) {
#pragma unroll
    for (int j = 0; j < N; j++) q.w[j] = __float_as_uint((float)x[j]);
  }
};
template <>
struct ga__lm_type<ga_double> {
  template <int N, typename F>
  static __device__ __forceinline__ void get(F x[N], const ga__lm_raw<8 * N> &q) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const unsigned long long u = (unsigned long long)q.w[2 * j + 1] << 32 | q.w[2 * j];
      double d;
      memcpy(&d, &u, 8);
      x[j] = (F)d;
    }
  }
  template <int N, typename F>
  static __device__ __forceinline__ void put(ga__lm_raw<8 * N> &q, const F x[N]) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const double d = (double)x[j];
      unsigned long long u;
      memcpy(&u, &d, 8);
      q.w[2 * j] = (unsigned int)u;
      q.w[2 * j + 1] = (unsigned int)(u >> 32);
    }
  }
};
template <typename T, int N, typename F>
static __device__ __forceinline__ void ga__lm_get(F x[N], const ga__lm_vec<T, N> &q) {
  ga__lm_type<T>::template get<N, F>(x, q);
}
template <typename T, int N, typename F>
static __device__ __forceinline__ void ga__lm_put(ga__lm_vec<T, N> &q, const F x[N]) {
  ga__lm_type<T>::template put<N, F>(q, x);
}

#define GA_LM_MAXD 4

/* Byte offset of leading index i: the dimensions left after collapsing, last one fastest. Quotients
 * of 32-bit numbers are several times cheaper; an index of 32 bits is below 2^32 - 1, which stands for
 * any longer dimension. */
template <int ND>
static __device__ __forceinline__ long long ga__lm_offset(unsigned int i, const unsigned long long *dims,
                                                          const long long *strs) {
  long long p = 0;
#pragma unroll
  for (int d = ND - 1; d > 0; d--) {
    const unsigned int n = dims[d] > 0xffffffffULL ? 0xffffffffu : (unsigned int)dims[d];
    const unsigned int q = i / n;
    p += (long long)(i - q * n) * strs[d];
    i = q;
  }
  return p + (long long)i * strs[0];
}
template <int ND>
static __device__ __forceinline__ long long ga__lm_offset(unsigned long long i,
                                                          const unsigned long long *dims,
                                                          const long long *strs) {
  if (ND <= 1) return (long long)i * strs[0];
  if (i < 0xffffffffULL) return ga__lm_offset<ND>((unsigned int)i, dims, strs);
  long long p = 0;
#pragma unroll
  for (int d = ND - 1; d > 0; d--) {
    const unsigned long long q = i / dims[d];
    p += (long long)(i - q * dims[d]) * strs[d];
    i = q;
  }
  return p + (long long)i * strs[0];
}
#endif
