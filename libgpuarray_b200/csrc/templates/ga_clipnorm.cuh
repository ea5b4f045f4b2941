/* The norm over a list of arrays, and the arrays scaled by what the norm says.
 *
 *   norm = |scale| * sqrt(sum over all arrays and elements of x^2)
 *   dst  = src * scale * (norm > limit ? limit / norm : 1)      (NaN norm: NaN)
 *
 * Both kernels walk the arrays as one sequence of blocks of GA_CN_VECS 16-byte
 * vectors; a block finds its array by halving over the arrays' first blocks in
 * the parameter block. Bound by memory: the arrays are read once for the norm;
 * the second pass goes through the blocks backwards, so that what the first
 * one read last is read from L2, and writes once.
 *
 * Defines needed: GA_CN_CAP (entries of the table). */
#include "ga_lm_common.cuh"

#define GA_CN_THREADS 256
#define GA_CN_VECS 2048u /* vectors of a block: 8 per thread */

struct ga__cn_item {
  const char *src;
  char *dst;
  unsigned long long n;
  unsigned int first; /* its first block */
  short stype, dtype; /* 0 half, 1 float, 2 double */
};
struct ga__cn_layout {
  unsigned int count, blocks;
  unsigned int slot;  /* first partial of this launch */
  unsigned int slots; /* partials of all launches if this is the last one, else 0 */
  double scale, limit;
  ga__cn_item item[GA_CN_CAP];
};
/* what the norm kernel leaves for the scaling one */
struct ga__cn_result {
  double factor;
  unsigned int ticket;
};

static __device__ __forceinline__ unsigned int ga__cn_find(const ga__cn_layout &L, unsigned int b) {
  unsigned int lo = 0, hi = L.count; /* item[lo].first <= b < item[hi].first */
  while (hi - lo > 1) {
    const unsigned int mid = (lo + hi) / 2;
    if (L.item[mid].first <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

/* A block of an array: 8 vectors of a thread. */
#define GA_CN_U 8
struct ga__cn_at {
  const ga__cn_item *t;
  unsigned int skip;     /* elements of the first vector below the array's start */
  unsigned long long w0; /* the thread's first vector */
  int inner;             /* every vector of the block is whole */
};

template <int ES>
static __device__ __forceinline__ ga__cn_at ga__cn_open(const ga__cn_item &t, unsigned int b) {
  const unsigned int E = 16 / ES;
  ga__cn_at a;
  const unsigned long long w = (unsigned long long)(b - t.first) * GA_CN_VECS;
  a.t = &t;
  a.skip = (unsigned int)((size_t)t.src & 15) / ES;
  a.w0 = w + threadIdx.x;
  a.inner = w * E >= a.skip && (w + GA_CN_VECS) * E - a.skip <= t.n;
  return a;
}

/* The thread's vectors; elements outside the array read as 0. */
template <int ES>
static __device__ __forceinline__ void ga__cn_load(ga__lm_raw<16> q[GA_CN_U], const ga__cn_at &a) {
  const unsigned int E = 16 / ES;
  const char *base = a.t->src - a.skip * ES; /* on a 16-byte boundary */
  if (a.inner) {
#pragma unroll
    for (int u = 0; u < GA_CN_U; u++)
      q[u] = ga__lm_load<ga__lm_raw<16> >(base + (a.w0 + u * GA_CN_THREADS) * 16);
    return;
  }
#pragma unroll
  for (int u = 0; u < GA_CN_U; u++) {
    const unsigned long long w = a.w0 + u * GA_CN_THREADS, i = w * E - a.skip; /* wraps below the start */
    if (w * E >= a.skip && i + E <= a.t->n) {
      q[u] = ga__lm_load<ga__lm_raw<16> >(base + w * 16);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) q[u].w[j] = 0;
#pragma unroll
    for (int j = 0; j < (int)E; j++)
      if (i + j < a.t->n) {
        const ga__lm_raw<ES> one = ga__lm_load<ga__lm_raw<ES> >(a.t->src + (i + j) * ES);
        if (ES == 2) q[u].w[j / 2] |= (unsigned int)one.w[0] << (16 * (j & 1));
        else
          for (int h = 0; h < (ES < 4 ? 1 : ES / 4); h++) q[u].w[j * (ES / 4) + h] = one.w[h];
      }
  }
}

/* Squares of a vector, summed in float pairs: those of halfs are exact and 8 of them are summed
 * before they go to double; floats and doubles are squared in double, so that no finite value
 * overflows or vanishes. */
static __device__ __forceinline__ double ga__cn_squares(const ga__lm_raw<16> &q, ga_half) {
  ga__f2 s = ga__f2_of(0.0f, 0.0f);
  float a, b;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    ga__unpack_h2(q.w[j], a, b);
    const ga__f2 x = ga__f2_of(a, b);
    s = ga__f2_fma(x, x, s);
  }
  ga__f2_to(s, a, b);
  return (double)(a + b);
}
static __device__ __forceinline__ double ga__cn_squares(const ga__lm_raw<16> &q, ga_float) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const double x = (double)__uint_as_float(q.w[j]);
    s = fma(x, x, s);
  }
  return s;
}
static __device__ __forceinline__ double ga__cn_squares(const ga__lm_raw<16> &q, ga_double) {
  double x[2];
  ga__lm_get<ga_double, 2>(x, q);
  return fma(x[1], x[1], x[0] * x[0]);
}

template <typename T>
static __device__ __forceinline__ double ga__cn_block(const ga__cn_item &t, unsigned int b) {
  ga__lm_raw<16> q[GA_CN_U];
  ga__cn_load<(int)sizeof(T)>(q, ga__cn_open<(int)sizeof(T)>(t, b));
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < GA_CN_U; u++) s += ga__cn_squares(q[u], T());
  return s;
}

extern "C" __global__ void __launch_bounds__(GA_CN_THREADS)
ga_cn_norm(const __grid_constant__ ga__cn_layout L, double *part, ga__cn_result *res, char *norm,
           int norm_is_double) {
  ga__grid_dependency_sync();
  __shared__ double warps[GA_CN_THREADS / 32];
  __shared__ int last;
  double s = 0.0;
  for (unsigned int b = blockIdx.x; b < L.blocks; b += gridDim.x) {
    const ga__cn_item &t = L.item[ga__cn_find(L, b)];
    if (t.stype == 0) s += ga__cn_block<ga_half>(t, b);
    else if (t.stype == 1) s += ga__cn_block<ga_float>(t, b);
    else s += ga__cn_block<ga_double>(t, b);
  }
  const unsigned int lane = threadIdx.x % 32;
#pragma unroll
  for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (lane == 0) warps[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < GA_CN_THREADS / 32; i++) s += warps[i];
    part[L.slot + blockIdx.x] = s;
    last = 0;
    if (L.slots != 0) {
      __threadfence();
      last = atomicAdd(&res->ticket, 1u) == gridDim.x - 1;
      __threadfence();
    }
  }
  __syncthreads();
  if (!last) return;
  /* the last CTA of the last launch adds the partials, always in the same order */
  s = 0.0;
  for (unsigned int i = threadIdx.x; i < L.slots; i += GA_CN_THREADS) s += __ldcg(&part[i]);
#pragma unroll
  for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
  __syncthreads();
  if (lane == 0) warps[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < GA_CN_THREADS / 32; i++) s += warps[i];
    const double size = sqrt(s), v = size * fabs(L.scale);
    res->ticket = 0;
    /* scale * limit / v without the scale, whose product with the size need not be a double */
    res->factor = v != v ? v : (v > L.limit ? copysign(L.limit / size, L.scale) : L.scale);
    if (norm_is_double) *reinterpret_cast<double *>(norm) = v;
    else *reinterpret_cast<float *>(norm) = (float)v;
  }
}

/* Halfs and floats times a factor that no normal float holds, as that of large gradients and a small
 * limit: elements and results may be ordinary floats all the same, so products are taken in double.
 * An element at a time, apart from the loops below, which it would make slower (0.7 % on 295 M halfs). */
static __device__ __forceinline__ void ga__cn_scale_wide(const ga__cn_item &t, unsigned int b, double factor) {
  const unsigned int E = t.stype == 0 ? 8 : 4, es = 16 / E, skip = (unsigned int)((size_t)t.src & 15) / es;
  const unsigned long long first = (unsigned long long)(b - t.first) * GA_CN_VECS * E;
  for (unsigned int k = threadIdx.x; k < GA_CN_VECS * E; k += GA_CN_THREADS) {
    const unsigned long long i = first + k - skip; /* wraps below the start */
    if (i >= t.n) continue;
    float x;
    if (t.stype == 0) x = ga_half2float(*reinterpret_cast<const ga_half *>(t.src + i * 2));
    else x = *reinterpret_cast<const float *>(t.src + i * 4);
    const double y = (double)x * factor;
    if (t.dtype == 0) *reinterpret_cast<unsigned short *>(t.dst + i * 2) = ga__half_bits(y);
    else *reinterpret_cast<float *>(t.dst + i * 4) = (float)y;
  }
}

template <typename T, typename D, typename F>
static __device__ __forceinline__ void ga__cn_scale(const ga__cn_item &t, unsigned int b, F factor) {
  const int E = 16 / (int)sizeof(T);
  typedef ga__lm_vec<D, E> vec;
  const ga__cn_at a = ga__cn_open<(int)sizeof(T)>(t, b);
  char *base = t.dst - a.skip * sizeof(D);
  const int aligned = ((size_t)base & (alignof(vec) - 1)) == 0;
  ga__lm_raw<16> q[GA_CN_U];
  ga__cn_load<(int)sizeof(T)>(q, a);
#pragma unroll
  for (int u = 0; u < GA_CN_U; u++) {
    const unsigned long long w = a.w0 + u * GA_CN_THREADS, i = w * E - a.skip;
    F x[E];
    ga__lm_get<T, E>(x, q[u]);
#pragma unroll
    for (int j = 0; j < E; j++) x[j] *= factor;
    if (aligned && (a.inner || (w * E >= a.skip && i + E <= t.n))) {
      vec o;
      ga__lm_put<D, E>(o, x);
      ga__lm_store(base + w * sizeof(vec), o);
    } else {
#pragma unroll
      for (int j = 0; j < E; j++)
        if (i + j < t.n) {
          ga__lm_vec<D, 1> o;
          ga__lm_put<D, 1>(o, x + j);
          ga__lm_store(t.dst + (i + j) * sizeof(D), o);
        }
    }
  }
}

/* A block for each CTA, not a fixed share of the blocks: the SMs are not equally fast. */
extern "C" __global__ void __launch_bounds__(GA_CN_THREADS)
ga_cn_scale(const __grid_constant__ ga__cn_layout L, const ga__cn_result *res) {
  ga__grid_dependency_sync();
  const double factor = __ldcg(&res->factor);
  const float f = (float)factor;
  const unsigned int b = L.blocks - 1 - blockIdx.x;
  const ga__cn_item &t = L.item[ga__cn_find(L, b)];
  /* an array that stays where it is and is multiplied by one is what it was */
  if (t.dst == t.src && t.stype == t.dtype && factor == 1.0) return;
  const double size = fabs(factor); /* zero, after an infinite norm or for a limit of 0, is a float */
  if (t.stype != 2 && size != 0.0 && (size < 1.1754943508222875e-38 || size > 3.4028234663852886e38))
    return ga__cn_scale_wide(t, b, factor);
  if (t.stype == 0) {
    if (t.dtype == 0) ga__cn_scale<ga_half, ga_half, float>(t, b, f);
    else ga__cn_scale<ga_half, ga_float, float>(t, b, f);
  } else if (t.stype == 1) {
    ga__cn_scale<ga_float, ga_float, float>(t, b, f);
  } else {
    ga__cn_scale<ga_double, ga_double, double>(t, b, factor);
  }
}
