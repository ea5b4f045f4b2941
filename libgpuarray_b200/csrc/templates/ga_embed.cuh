/* Token embedding: rows of a table by id, and the sum of rows by id.
 *
 *   ga_embed:     out[t, :] = scale * table[row(ids[t]), :]
 *   gradient:     dtable[v, :] (+)= scale * sum over {t : row(ids[t]) = v} of dout[t, :]
 *
 * row(i) = i, or i + V for negative i (the rule of GpuArray_take1); the padding
 * id gives a row of zeros and contributes nothing to the gradient; an id
 * outside the table is skipped and reported through *err.
 *
 * Defines needed: GA_EM_BUILD_LOOKUP or GA_EM_BUILD_GRAD, GA_EM_A_T (table, or
 * dout), GA_EM_O_T (out, or dtable), GA_EM_I_T (ids), GA_EM_F_T (arithmetic),
 * GA_EM_E (elements of a vector), GA_EM_ND (leading dimensions). */
#include "ga_lm_common.cuh"

struct ga__em_layout {
  unsigned long long n;      /* tokens */
  unsigned long long v;      /* table rows */
  unsigned int nv;           /* vectors of GA_EM_E elements in a row */
  unsigned int chunk;        /* gradient: sorted tokens summed by one group of threads */
  unsigned int chunks;
  int has_pad;
  long long pad;
  double scale;
  unsigned long long dims[GA_LM_MAXD];
  long long i_str[GA_LM_MAXD];
  long long t_str[GA_LM_MAXD]; /* of out (lookup) or dout (gradient), by token */
  long long t_col, v_row, v_col; /* its element stride; the table's (dtable's) row and element stride */
};

/* Table row of token i's id, or -1 for the padding id, -2 for an id outside the table. */
static __device__ __forceinline__ long long ga__em_row(const ga__em_layout &L, const char *ids,
                                                       unsigned long long i) {
  const GA_EM_I_T raw =
      *reinterpret_cast<const GA_EM_I_T *>(ids + ga__lm_offset<GA_EM_ND>(i, L.dims, L.i_str));
  long long r = (long long)raw;
  if (L.has_pad && r == L.pad) return -1;
  /* an unsigned 64-bit id of 2^63 and more is outside any table, not a negative number */
  if (r < 0 && (GA_EM_I_T)-1 > (GA_EM_I_T)0) return -2;
  if (r < 0) r += (long long)L.v;
  return r < 0 || r >= (long long)L.v ? -2 : r;
}

template <typename T>
static __device__ __forceinline__ void ga__em_load(GA_EM_F_T x[GA_EM_E], const char *p, long long col) {
  if (GA_EM_E == 1) {
    x[0] = (GA_EM_F_T)ga__lm_get(*reinterpret_cast<const T *>(p));
  } else {
    const ga__lm_vec<T, GA_EM_E> q = *reinterpret_cast<const ga__lm_vec<T, GA_EM_E> *>(p);
#pragma unroll
    for (int j = 0; j < GA_EM_E; j++) x[j] = (GA_EM_F_T)ga__lm_get(q.v[j]);
  }
}

#ifdef GA_EM_BUILD_LOOKUP
#define GA_EM_U 4
/* A thread owns one vector position of the row and GA_EM_U tokens, so that
 * GA_EM_U independent loads are in flight behind one round trip for the ids.
 * Bound by memory: a row is read once per token (tokens that repeat find it in
 * L2) and written once. */
extern "C" __global__ void __launch_bounds__(256)
ga_embed(const __grid_constant__ ga__em_layout L, char *out, const char *table, const char *ids,
         int *err) {
  ga__grid_dependency_sync();
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
  const unsigned long long t0 =
      ((unsigned long long)blockIdx.x * blockDim.y + threadIdx.y) * GA_EM_U;
  if (v >= L.nv || t0 >= L.n) return;
  const GA_EM_F_T scale = (GA_EM_F_T)L.scale;
  long long row[GA_EM_U];
#pragma unroll
  for (int u = 0; u < GA_EM_U; u++) row[u] = t0 + u < L.n ? ga__em_row(L, ids, t0 + u) : -3;
  GA_EM_F_T x[GA_EM_U][GA_EM_E];
#pragma unroll
  for (int u = 0; u < GA_EM_U; u++) {
#pragma unroll
    for (int j = 0; j < GA_EM_E; j++) x[u][j] = 0;
    if (row[u] >= 0)
      ga__em_load<GA_EM_A_T>(x[u], table + row[u] * L.v_row + (long long)v * GA_EM_E * L.v_col, L.v_col);
  }
#pragma unroll
  for (int u = 0; u < GA_EM_U; u++) {
    if (row[u] == -2 && v == 0 && err != nullptr) *err = -1;
    if (row[u] < -1) continue;
    char *p = out + ga__lm_offset<GA_EM_ND>(t0 + u, L.dims, L.t_str) + (long long)v * GA_EM_E * L.t_col;
    ga__lm_vec<GA_EM_O_T, GA_EM_E> q;
#pragma unroll
    for (int j = 0; j < GA_EM_E; j++) ga__lm_put(&q.v[j], x[u][j] * scale);
    *reinterpret_cast<ga__lm_vec<GA_EM_O_T, GA_EM_E> *>(p) = q;
  }
}
#endif

#ifdef GA_EM_BUILD_GRAD
/* The gradient is a sum over SORTED tokens: three launches that depend on
 * nothing but the ids' values, so that the result is the same bits every time.
 *
 * 1. ga_eg_order: order[rank] = token, key[rank] = row, by row and, within a
 *    row, by token. Tokens that contribute nothing get the key V and go last.
 * 2. ga_eg_sum: the sorted tokens are cut into equal chunks; a group of threads
 *    sums a chunk's rows, one vector position per thread. A run of equal keys
 *    that lies inside the chunk is finished and written; the parts of runs that
 *    cross a chunk's ends go to `part`, which holds two rows per chunk.
 * 3. ga_eg_join: the group of the chunk in which a crossing run starts adds its
 *    parts in order and writes the row.
 * Rows that no token names are written by ga_eg_zero before (unless the
 * gradient is accumulated). */

/* The tokens' ranks by counting: a warp per token compares its key with all. */
extern "C" __global__ void __launch_bounds__(256)
ga_eg_order(const __grid_constant__ ga__em_layout L, unsigned int *key, unsigned int *order,
            const char *ids, int *err) {
  ga__grid_dependency_sync();
  const unsigned int n = (unsigned int)L.n, lane = threadIdx.x % 32;
  const unsigned int t = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (t >= n) return; /* a whole warp */
  const long long mine = ga__em_row(L, ids, t);
  if (mine == -2 && lane == 0 && err != nullptr) *err = -1;
  const unsigned long long k = mine < 0 ? L.v : (unsigned long long)mine;
  unsigned int before = 0;
  for (unsigned int i = lane; i < n; i += 32) {
    const long long other = ga__em_row(L, ids, i);
    const unsigned long long o = other < 0 ? L.v : (unsigned long long)other;
    before += o < k || (o == k && i < t);
  }
  before = ga__warp_sum_u32(before);
  if (lane == 0) {
    key[before] = (unsigned int)k;
    order[before] = t;
  }
}

extern "C" __global__ void __launch_bounds__(256)
ga_eg_zero(const __grid_constant__ ga__em_layout L, char *dtable) {
  ga__grid_dependency_sync();
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
  if (v >= L.nv) return;
  for (unsigned long long r = (unsigned long long)blockIdx.x * blockDim.y + threadIdx.y; r < L.v;
       r += (unsigned long long)gridDim.x * blockDim.y) {
    ga__lm_vec<GA_EM_O_T, GA_EM_E> q;
#pragma unroll
    for (int j = 0; j < GA_EM_E; j++) ga__lm_put(&q.v[j], (GA_EM_F_T)0);
    *reinterpret_cast<ga__lm_vec<GA_EM_O_T, GA_EM_E> *>(dtable + (long long)r * L.v_row +
                                                       (long long)v * GA_EM_E * L.v_col) = q;
  }
}

static __device__ __forceinline__ void ga__eg_write(const ga__em_layout &L, char *dtable,
                                                    unsigned int row, unsigned int v,
                                                    const GA_EM_F_T acc[GA_EM_E]) {
  const GA_EM_F_T scale = (GA_EM_F_T)L.scale;
  char *p = dtable + (long long)row * L.v_row + (long long)v * GA_EM_E * L.v_col;
  ga__lm_vec<GA_EM_O_T, GA_EM_E> q;
#if GA_EM_ACCUMULATE
  GA_EM_F_T old[GA_EM_E];
  ga__em_load<GA_EM_O_T>(old, p, L.v_col);
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) ga__lm_put(&q.v[j], old[j] + acc[j] * scale);
#else
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) ga__lm_put(&q.v[j], acc[j] * scale);
#endif
  *reinterpret_cast<ga__lm_vec<GA_EM_O_T, GA_EM_E> *>(p) = q;
}

#define GA_EG_U 8

static __device__ __forceinline__ void ga__eg_park(GA_EM_F_T *part, unsigned long long slot,
                                                   unsigned int nv, unsigned int v,
                                                   const GA_EM_F_T acc[GA_EM_E]) {
  GA_EM_F_T *p = part + (slot * nv + v) * GA_EM_E;
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) p[j] = acc[j];
}

extern "C" __global__ void __launch_bounds__(256)
ga_eg_sum(const __grid_constant__ ga__em_layout L, char *dtable, const char *dout,
          const unsigned int *key, const unsigned int *order, GA_EM_F_T *part) {
  ga__grid_dependency_sync();
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
  const unsigned int c = blockIdx.x * blockDim.y + threadIdx.y;
  if (v >= L.nv || c >= L.chunks) return;
  const unsigned int n = (unsigned int)L.n;
  const unsigned int lo = c * L.chunk, hi = n - lo < L.chunk ? n : lo + L.chunk;
  const unsigned int none = (unsigned int)L.v;
  unsigned int cur = key[lo];
  int open_head = lo > 0 && key[lo - 1] == cur; /* the run began in an earlier chunk */
  GA_EM_F_T acc[GA_EM_E];
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) acc[j] = 0;
  for (unsigned int i = lo; i < hi && cur != none; i += GA_EG_U) {
    unsigned int k[GA_EG_U];
    GA_EM_F_T x[GA_EG_U][GA_EM_E];
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++) k[u] = i + u < hi ? key[i + u] : none;
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++)
      if (k[u] != none)
        ga__em_load<GA_EM_A_T>(x[u],
                               dout + ga__lm_offset<GA_EM_ND>(order[i + u], L.dims, L.t_str) +
                                   (long long)v * GA_EM_E * L.t_col,
                               L.t_col);
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++) {
      if (i + u >= hi) break;
      if (k[u] != cur) { /* the run ends inside the chunk */
        if (open_head) ga__eg_park(part, 2ULL * c, L.nv, v, acc);
        else ga__eg_write(L, dtable, cur, v, acc);
        open_head = 0;
        cur = k[u];
#pragma unroll
        for (int j = 0; j < GA_EM_E; j++) acc[j] = 0;
        if (cur == none) break;
      }
#pragma unroll
      for (int j = 0; j < GA_EM_E; j++) acc[j] += x[u][j];
    }
  }
  if (cur == none) return;
  if (open_head) ga__eg_park(part, 2ULL * c, L.nv, v, acc);
  else if (hi < n && key[hi] == cur) ga__eg_park(part, 2ULL * c + 1, L.nv, v, acc);
  else ga__eg_write(L, dtable, cur, v, acc);
}

extern "C" __global__ void __launch_bounds__(256)
ga_eg_join(const __grid_constant__ ga__em_layout L, char *dtable, const unsigned int *key,
           const GA_EM_F_T *part) {
  ga__grid_dependency_sync();
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
  const unsigned int c = blockIdx.x * blockDim.y + threadIdx.y;
  if (v >= L.nv || c + 1 >= L.chunks) return;
  const unsigned int lo = c * L.chunk, next = lo + L.chunk; /* next < n: chunk c + 1 exists */
  const unsigned int cur = key[next];
  /* only the chunk in which a crossing run starts joins it */
  if (cur == (unsigned int)L.v || key[next - 1] != cur) return;
  if (key[lo] == cur && lo > 0 && key[lo - 1] == cur) return;
  GA_EM_F_T acc[GA_EM_E];
  const GA_EM_F_T *p = part + ((2ULL * c + 1) * L.nv + v) * GA_EM_E;
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) acc[j] = p[j];
  for (unsigned int d = c + 1; d < L.chunks && key[d * L.chunk] == cur; d++) {
    p = part + (2ULL * d * L.nv + v) * GA_EM_E;
#pragma unroll
    for (int j = 0; j < GA_EM_E; j++) acc[j] += p[j];
  }
  ga__eg_write(L, dtable, cur, v, acc);
}
#endif
