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

/* Vector w of an array: elements w * E - skip ..., those inside [0, n); the others read as 0. */
template <typename T, int E>
static __device__ __forceinline__ ga__lm_vec<T, E> ga__cn_load(const char *src, unsigned long long n,
                                                               unsigned int skip,
                                                               unsigned long long w) {
  const unsigned long long i0 = w * E - skip; /* wraps below the start */
  if (w * E >= skip && i0 + E <= n)
    return *reinterpret_cast<const ga__lm_vec<T, E> *>(src + (long long)i0 * (long long)sizeof(T));
  ga__lm_vec<T, E> q;
#pragma unroll
  for (int j = 0; j < E; j++) {
    q.v[j] = T();
    if (i0 + j < n) q.v[j] = reinterpret_cast<const T *>(src)[i0 + j];
  }
  return q;
}

/* squares of one vector: exact in float for halves, summed over 8 of them before they go to
 * double; floats and doubles are squared in double, so that no finite value overflows or vanishes */
static __device__ __forceinline__ double ga__cn_squares(const ga__lm_vec<ga_half, 8> &q) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float x = ga_half2float(q.v[j]);
    s = fmaf(x, x, s);
  }
  return (double)s;
}
template <typename T, int E>
static __device__ __forceinline__ double ga__cn_squares(const ga__lm_vec<T, E> &q) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < E; j++) s = fma((double)q.v[j], (double)q.v[j], s);
  return s;
}

#define GA_CN_U 8
template <typename T, int E>
static __device__ __forceinline__ double ga__cn_block(const ga__cn_item &t, unsigned int b) {
  const unsigned int skip = (unsigned int)((size_t)t.src & 15) / (unsigned int)sizeof(T);
  const unsigned long long w0 = (unsigned long long)(b - t.first) * GA_CN_VECS + threadIdx.x;
  ga__lm_vec<T, E> q[GA_CN_U];
#pragma unroll
  for (int u = 0; u < GA_CN_U; u++) q[u] = ga__cn_load<T, E>(t.src, t.n, skip, w0 + u * GA_CN_THREADS);
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < GA_CN_U; u++) s += ga__cn_squares(q[u]);
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
    if (t.stype == 0) s += ga__cn_block<ga_half, 8>(t, b);
    else if (t.stype == 1) s += ga__cn_block<ga_float, 4>(t, b);
    else s += ga__cn_block<ga_double, 2>(t, b);
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
    const double v = sqrt(s) * fabs(L.scale);
    res->ticket = 0;
    res->factor = v != v ? v : (v > L.limit ? L.scale * (L.limit / v) : L.scale);
    if (norm_is_double) *reinterpret_cast<double *>(norm) = v;
    else *reinterpret_cast<float *>(norm) = (float)v;
  }
}

template <typename T, typename D, typename F, int E>
static __device__ __forceinline__ void ga__cn_scale(const ga__cn_item &t, unsigned int b, F factor) {
  const unsigned int skip = (unsigned int)((size_t)t.src & 15) / (unsigned int)sizeof(T);
  const unsigned long long w0 = (unsigned long long)(b - t.first) * GA_CN_VECS + threadIdx.x;
  typedef ga__lm_vec<D, E> vec;
  const int aligned = (((size_t)t.dst - (size_t)skip * sizeof(D)) & (alignof(vec) - 1)) == 0;
  ga__lm_vec<T, E> q[GA_CN_U];
#pragma unroll
  for (int u = 0; u < GA_CN_U; u++) q[u] = ga__cn_load<T, E>(t.src, t.n, skip, w0 + u * GA_CN_THREADS);
#pragma unroll
  for (int u = 0; u < GA_CN_U; u++) {
    const unsigned long long w = w0 + u * GA_CN_THREADS, i0 = w * E - skip;
    vec o;
#pragma unroll
    for (int j = 0; j < E; j++) ga__lm_put(&o.v[j], (F)ga__lm_get(q[u].v[j]) * factor);
    if (aligned && w * E >= skip && i0 + E <= t.n) {
      *reinterpret_cast<vec *>(t.dst + (long long)i0 * (long long)sizeof(D)) = o;
    } else {
#pragma unroll
      for (int j = 0; j < E; j++)
        if (i0 + j < t.n) reinterpret_cast<D *>(t.dst)[i0 + j] = o.v[j];
    }
  }
}

extern "C" __global__ void __launch_bounds__(GA_CN_THREADS)
ga_cn_scale(const __grid_constant__ ga__cn_layout L, const ga__cn_result *res) {
  ga__grid_dependency_sync();
  const double factor = __ldcg(&res->factor);
  const float f = (float)factor;
  for (unsigned int i = blockIdx.x; i < L.blocks; i += gridDim.x) {
    const unsigned int b = L.blocks - 1 - i;
    const ga__cn_item &t = L.item[ga__cn_find(L, b)];
    /* an array that stays where it is and is multiplied by one is what it was */
    if (t.dst == t.src && t.stype == t.dtype && factor == 1.0) continue;
    if (t.stype == 0) {
      if (t.dtype == 0) ga__cn_scale<ga_half, ga_half, float, 8>(t, b, f);
      else ga__cn_scale<ga_half, ga_float, float, 8>(t, b, f);
    } else if (t.stype == 1) {
      ga__cn_scale<ga_float, ga_float, float, 4>(t, b, f);
    } else {
      ga__cn_scale<ga_double, ga_double, double, 2>(t, b, factor);
    }
  }
}
