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
 * GA_EM_E (elements of a vector), GA_EM_C (vectors of a thread), GA_EM_ND
 * (leading dimensions). */
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

/* Table row of token i's id, or -1 for the padding id, -2 for an id outside the table. The lookup
 * counts tokens in 64 bits, the gradient (up to 2^31 - 1 of them) in 32. */
template <typename I>
static __device__ __forceinline__ long long ga__em_row(const ga__em_layout &L, const char *ids, I i) {
  const GA_EM_I_T raw =
      *reinterpret_cast<const GA_EM_I_T *>(ids + ga__lm_offset<GA_EM_ND>(i, L.dims, L.i_str));
  long long r = (long long)raw;
  if (L.has_pad && r == L.pad) return -1;
  /* an unsigned 64-bit id of 2^63 and more is outside any table, not a negative number */
  if (r < 0 && (GA_EM_I_T)-1 > (GA_EM_I_T)0) return -2;
  if (r < 0) r += (long long)L.v;
  return r < 0 || r >= (long long)L.v ? -2 : r;
}

/* A thread's part of a row: GA_EM_C vectors of GA_EM_E elements, blockDim.x vectors apart. Rows
 * that start off the boundary of a 16-byte vector are moved in narrower ones; several of them in
 * one thread keep as many bytes in flight. */
#define GA_EM_N (GA_EM_E * GA_EM_C)
typedef ga__lm_vec<GA_EM_A_T, GA_EM_E> ga__em_in1;
typedef ga__lm_vec<GA_EM_O_T, GA_EM_E> ga__em_out1;
struct ga__em_in {
  ga__em_in1 c[GA_EM_C];
};
struct ga__em_out {
  ga__em_out1 c[GA_EM_C];
};
struct ga__em_pos {
  unsigned int v; /* the first vector's position; some of the others may lie beyond the row */
  unsigned int nv;
};
static __device__ __forceinline__ ga__em_pos ga__em_here(const ga__em_layout &L) {
  ga__em_pos p;
  p.v = blockIdx.y * blockDim.x * GA_EM_C + threadIdx.x;
  p.nv = L.nv;
  return p;
}
template <typename V, typename R>
static __device__ __forceinline__ V ga__em_read(const char *row, long long col, ga__em_pos p) {
  V q;
#pragma unroll
  for (int c = 0; c < GA_EM_C; c++) {
    const unsigned int v = p.v + c * blockDim.x;
    if (c == 0 || v < p.nv)
      q.c[c] = ga__lm_load<R>(row + (long long)v * GA_EM_E * col);
  }
  return q;
}
static __device__ __forceinline__ void ga__em_write(char *row, long long col, ga__em_pos p,
                                                    const ga__em_out &q) {
#pragma unroll
  for (int c = 0; c < GA_EM_C; c++) {
    const unsigned int v = p.v + c * blockDim.x;
    if (c == 0 || v < p.nv) ga__lm_store(row + (long long)v * GA_EM_E * col, q.c[c]);
  }
}
template <typename T, typename V>
static __device__ __forceinline__ void ga__em_get(GA_EM_F_T x[GA_EM_N], const V &q) {
#pragma unroll
  for (int c = 0; c < GA_EM_C; c++) ga__lm_get<T, GA_EM_E>(x + c * GA_EM_E, q.c[c]);
}
static __device__ __forceinline__ void ga__em_put(ga__em_out &q, const GA_EM_F_T x[GA_EM_N]) {
#pragma unroll
  for (int c = 0; c < GA_EM_C; c++) ga__lm_put<GA_EM_O_T, GA_EM_E>(q.c[c], x + c * GA_EM_E);
}
template <typename V>
static __device__ __forceinline__ V ga__em_zero() {
  V q;
#pragma unroll
  for (int c = 0; c < GA_EM_C; c++)
#pragma unroll
    for (int j = 0; j < (int)(sizeof(q.c[c].w) / sizeof(q.c[c].w[0])); j++) q.c[c].w[j] = 0;
  return q;
}

#ifdef GA_EM_BUILD_LOOKUP
/* loads of a thread in flight (4 x 4095 tokens of 4096 halfs: 34 us with 4, 35 with 8, 42 with 16) */
#define GA_EM_U 4
#define GA_EM_TOKENS 256 /* of a CTA's groups at most */
#define GA_EM_NOWHERE (-0x7fffffffffffffffLL) /* no offset of an array */
/* A group of threads (blockIdx.x, threadIdx.y) owns L.chunk tokens and one slice of their rows, a
 * vector position per thread. It first finds the tokens' rows and places together, a token per
 * thread, so that neither the ids' round trip nor the divisions of their dimensions come with
 * every vector; then GA_EM_U rows at a time are in flight.
 * Bound by memory: a row is read once per token (tokens that repeat find it in L2) and written
 * once. */
extern "C" __global__ void __launch_bounds__(256)
ga_embed(const __grid_constant__ ga__em_layout L, char *out, const char *table, const char *ids,
         int *err) {
  ga__grid_dependency_sync();
  __shared__ long long from[GA_EM_TOKENS], to[GA_EM_TOKENS];
  const unsigned int tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  const unsigned long long first = (unsigned long long)blockIdx.x * blockDim.y * L.chunk;
  const unsigned int here = blockDim.y * L.chunk; /* tokens of all groups of this CTA */
  for (unsigned int i = tid; i < here; i += threads) {
    long long row = -2, place = 0;
    if (first + i < L.n) {
      row = ga__em_row(L, ids, first + i);
      place = ga__lm_offset<GA_EM_ND>(first + i, L.dims, L.t_str);
      if (row == -2 && blockIdx.y == 0 && err != nullptr) *err = -1;
    }
    from[i] = row < 0 ? GA_EM_NOWHERE : row * L.v_row; /* padding: nothing is read */
    to[i] = row < -1 ? GA_EM_NOWHERE : place;          /* no such row: nothing is written */
  }
  __syncthreads();
  const ga__em_pos at = ga__em_here(L);
  if (at.v >= L.nv) return;
  const GA_EM_F_T scale = (GA_EM_F_T)L.scale;
  const unsigned int t1 = (threadIdx.y + 1) * L.chunk;
  for (unsigned int t = threadIdx.y * L.chunk; t < t1; t += GA_EM_U) {
    ga__em_in q[GA_EM_U];
#pragma unroll
    for (int u = 0; u < GA_EM_U; u++) {
      q[u] = ga__em_zero<ga__em_in>();
      if (t + u < t1 && to[t + u] != GA_EM_NOWHERE && from[t + u] != GA_EM_NOWHERE)
        q[u] = ga__em_read<ga__em_in, ga__em_in1>(table + from[t + u], L.v_col, at);
    }
#pragma unroll
    for (int u = 0; u < GA_EM_U; u++) {
      if (t + u >= t1 || to[t + u] == GA_EM_NOWHERE) continue;
      GA_EM_F_T x[GA_EM_N];
      ga__em_get<GA_EM_A_T>(x, q[u]);
#pragma unroll
      for (int j = 0; j < GA_EM_N; j++) x[j] *= scale;
      ga__em_out o;
      ga__em_put(o, x);
      ga__em_write(out + to[t + u], L.t_col, at, o);
    }
  }
}
#endif

#ifdef GA_EM_BUILD_GRAD
#ifndef GA_EG_ROUNDS /* of the one-launch sort, and its CTAs */
#define GA_EG_ROUNDS 1
#define GA_EG_CLUSTER 1
#endif
/* The gradient is a sum over SORTED tokens, in launches that depend on nothing
 * but the ids' values, so that the result is the same bits every time.
 *
 * Few tokens: ga_eg_direct. A CTA owns a range of table rows and a slice of
 * their vectors, picks its tokens from all ids, sorts them in shared memory,
 * writes zeros and sums.
 *
 * More tokens: they are sorted by row and, within a row, by token (a radix sort
 * of GA_EG_BITS bits a pass), up to 32768 of them by one CTA or cluster in one
 * launch (ga_eg_sort_all), beyond by a ga_eg_count and a ga_eg_scatter for each
 * pass. Tokens that contribute nothing get the key V
 * and go last. ga_eg_zero writes zeros to all rows beside the sort.
 * Then ga_eg_sum: the sorted tokens are cut into equal chunks; a group of
 * threads sums a chunk's rows, one vector position per thread. A run of equal
 * keys that lies inside the chunk is finished and written; the parts of runs
 * that cross a chunk's ends are parked, two rows per chunk. ga_eg_join: the
 * group of the chunk in which a crossing run starts adds its parts in order
 * and writes the row. */

/* `old`: what the row holds so far, read ahead by the caller (used where it is added to) */
static __device__ __forceinline__ void ga__eg_write(const ga__em_layout &L, char *dtable,
                                                    unsigned int row, ga__em_pos at,
                                                    const GA_EM_F_T acc[GA_EM_N],
                                                    const ga__em_out &old) {
  const GA_EM_F_T scale = (GA_EM_F_T)L.scale;
  GA_EM_F_T x[GA_EM_N];
  ga__em_out q;
#if GA_EM_ACCUMULATE
  ga__em_get<GA_EM_O_T>(x, old);
#pragma unroll
  for (int j = 0; j < GA_EM_N; j++) x[j] += acc[j] * scale;
#else
#pragma unroll
  for (int j = 0; j < GA_EM_N; j++) x[j] = acc[j] * scale;
#endif
  ga__em_put(q, x);
  ga__em_write(dtable + (long long)row * L.v_row, L.v_col, at, q);
}
static __device__ __forceinline__ ga__em_out ga__eg_held(const ga__em_layout &L, const char *dtable,
                                                         unsigned int row, ga__em_pos at) {
  return ga__em_read<ga__em_out, ga__em_out1>(dtable + (long long)row * L.v_row, L.v_col, at);
}

/* Zeros for the rows, `bytes` of them where the rows are adjacent (0: row by row). One tile or
 * group of rows for each CTA: handed out one after the other they are written at 7.3 TB/s, by
 * CTAs that each walk a fixed share of the rows at 6.2 (the SMs are not equally fast).
 *
 * It runs beside the launch before it, whose CTAs sort: it does not wait for that one, which
 * itself released its successor only after waiting for all that came before. Its last CTA stays
 * until the sort is complete, so that whatever waits for this launch has waited for both. */
#define GA_EG_ZERO 512
extern "C" __global__ void __launch_bounds__(GA_EG_ZERO)
ga_eg_zero(const __grid_constant__ ga__em_layout L, char *dtable, unsigned long long bytes) {
  ga__grid_dependency_release();
  if (bytes > 0) {
    ga__lm_raw<16> q;
    q.w[0] = q.w[1] = q.w[2] = q.w[3] = 0;
    const unsigned long long at = ((unsigned long long)blockIdx.x * 4 * GA_EG_ZERO + threadIdx.x) * 16;
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (at + u * GA_EG_ZERO * 16 + 16 <= bytes) ga__lm_store(dtable + at + u * GA_EG_ZERO * 16, q);
    /* what is left is less than 16 bytes */
    const unsigned long long done = bytes / 16 * 16;
    if (blockIdx.x == 0 && threadIdx.x < bytes - done) dtable[done + threadIdx.x] = 0;
  } else {
    const unsigned int lane = threadIdx.x % 32, warps = GA_EG_ZERO / 32;
    for (unsigned long long r = (unsigned long long)blockIdx.x * warps + threadIdx.x / 32; r < L.v;
         r += (unsigned long long)gridDim.x * warps)
      for (unsigned int v = lane; v < L.nv; v += 32)
        ga__lm_store(dtable + (long long)r * L.v_row + (long long)v * GA_EM_E * L.v_col, ga__em_zero<ga__em_out>().c[0]);
  }
  if (blockIdx.x == gridDim.x - 1) ga__grid_dependency_wait();
}

/* ---- sorting ---- */
#define GA_EG_BITS 9
#define GA_EG_DIGITS (1 << GA_EG_BITS)
#define GA_EG_THREADS GA_EG_DIGITS /* a thread for each digit */
#define GA_EG_WARPS (GA_EG_THREADS / 32)
#define GA_EG_KEYS 4 /* a thread's keys of one round */
#define GA_EG_ROUND (GA_EG_THREADS * GA_EG_KEYS)

struct ga__eg_sort {
  unsigned int n;      /* tokens */
  unsigned int tiles;  /* CTAs that sort */
  unsigned int tile;   /* tokens of each, a multiple of GA_EG_ROUND */
  unsigned int passes; /* their number; this one's is `pass` */
  unsigned int pass;
};

static __device__ __forceinline__ unsigned int ga__eg_key(const ga__em_layout &L, const char *ids,
                                                          unsigned int i, int *err) {
  const long long r = ga__em_row(L, ids, i);
  if (r == -2 && err != nullptr) *err = -1;
  return r < 0 ? (unsigned int)L.v : (unsigned int)r;
}

/* Key i of a pass: the first pass makes them from the ids. */
static __device__ __forceinline__ unsigned int ga__eg_key_of(const ga__em_layout &L, const ga__eg_sort &S,
                                                             const char *ids, const unsigned int *key_in,
                                                             unsigned int i, int *err) {
  return S.pass == 0 ? ga__eg_key(L, ids, i, err) : key_in[i];
}

/* counts[digit][tile]: how many keys of a tile have the digit. (Counting for the next pass where
 * keys are scattered takes an atomic for each, thousands of them on the counts of a frequent id.) */
extern "C" __global__ void __launch_bounds__(GA_EG_THREADS)
ga_eg_count(const __grid_constant__ ga__em_layout L, const __grid_constant__ ga__eg_sort S,
            unsigned int *counts, const char *ids, const unsigned int *key_in, int *err) {
  ga__grid_dependency_sync();
  __shared__ unsigned int hist[GA_EG_DIGITS];
  const unsigned int d = threadIdx.x, tile = blockIdx.x;
  hist[d] = 0;
  __syncthreads();
  const unsigned int lo = tile * S.tile, hi = S.n - lo < S.tile ? S.n : lo + S.tile;
  for (unsigned int i = lo + threadIdx.x; i < hi; i += GA_EG_THREADS)
    atomicAdd(&hist[(ga__eg_key_of(L, S, ids, key_in, i, err) >> (S.pass * GA_EG_BITS)) & (GA_EG_DIGITS - 1)], 1u);
  __syncthreads();
  counts[d * S.tiles + tile] = hist[d];
}

/* The exclusive prefix of x over the CTA's GA_EG_THREADS threads. */
static __device__ __forceinline__ unsigned int ga__eg_prefix(unsigned int x, unsigned int sums[GA_EG_WARPS]) {
  const unsigned int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  unsigned int scan = x;
#pragma unroll
  for (int s = 1; s < 32; s *= 2) {
    const unsigned int o = __shfl_up_sync(0xffffffffu, scan, s);
    if (lane >= (unsigned int)s) scan += o;
  }
  if (lane == 31) sums[warp] = scan;
  __syncthreads();
  unsigned int r = scan - x;
  for (unsigned int w = 0; w < warp; w++) r += sums[w];
  return r;
}

/* Places of GA_EG_ROUND keys, GA_EG_KEYS of a thread: key j of a thread is key
 * (warp * GA_EG_KEYS + j) * 32 + lane of the round, there where `live` says so. A key goes behind
 * those of smaller digits and behind those of its own that stand before it. base: where the keys
 * of the digit that is this thread's number begin; it moves on. */
typedef unsigned int ga__eg_table[GA_EG_WARPS][GA_EG_DIGITS];
static __device__ __forceinline__ void ga__eg_places(const unsigned int digit[GA_EG_KEYS],
                                                     const int live[GA_EG_KEYS], unsigned int &base,
                                                     ga__eg_table &cnt, unsigned int at[GA_EG_KEYS]) {
  const unsigned int d = threadIdx.x, lane = d % 32, warp = d / 32;
#pragma unroll
  for (int w = 0; w < GA_EG_WARPS; w++) cnt[w][d] = 0;
  /* the lanes with a key's digit, from a vote for each of its bits (one match instruction takes
   * longer the more digits there are: a round 4 us, so 1.5) */
  unsigned int same[GA_EG_KEYS];
#pragma unroll
  for (int j = 0; j < GA_EG_KEYS; j++) {
    same[j] = __ballot_sync(0xffffffffu, live[j]);
#pragma unroll
    for (int b = 0; b < GA_EG_BITS; b++) {
      const int bit = (digit[j] >> b) & 1;
      const unsigned int set = __ballot_sync(0xffffffffu, bit);
      same[j] &= bit ? set : ~set;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < GA_EG_KEYS; j++) {
    const unsigned int seen = live[j] ? cnt[warp][digit[j]] : 0;
    at[j] = seen + __popc(same[j] & ((1u << lane) - 1));
    __syncwarp();
    if (live[j] && __ffs(same[j]) - 1 == (int)lane) cnt[warp][digit[j]] = seen + __popc(same[j]);
    __syncwarp();
  }
  __syncthreads();
  unsigned int x[GA_EG_WARPS];
#pragma unroll
  for (int w = 0; w < GA_EG_WARPS; w++) x[w] = cnt[w][d];
#pragma unroll
  for (int w = 0; w < GA_EG_WARPS; w++) { /* the digit's place for each warp */
    cnt[w][d] = base;
    base += x[w];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < GA_EG_KEYS; j++)
    if (live[j]) at[j] += cnt[warp][digit[j]];
}

/* One pass over many tokens. The first takes the ids themselves; the last leaves the byte offsets
 * of the tokens' rows of dout, so that the sums need no division. */
extern "C" __global__ void __launch_bounds__(GA_EG_THREADS)
ga_eg_scatter(const __grid_constant__ ga__em_layout L, const __grid_constant__ ga__eg_sort S,
              const unsigned int *counts, const char *ids,
              const unsigned int *key_in, const unsigned int *order_in, unsigned int *key,
              unsigned int *order, long long *off) {
  ga__grid_dependency_sync();
  __shared__ ga__eg_table cnt;
  __shared__ unsigned int sums[GA_EG_WARPS];
  const unsigned int d = threadIdx.x, lane = d % 32, warp = d / 32, tile = blockIdx.x;
  const unsigned int shift = S.pass * GA_EG_BITS;

  /* where the digit's keys of this tile begin */
  const unsigned int *c = counts + d * S.tiles;
  unsigned int total = 0, before = 0;
  for (unsigned int t = 0; t < S.tiles; t++) {
    const unsigned int x = c[t];
    total += x;
    before += t < tile ? x : 0;
  }
  unsigned int base = ga__eg_prefix(total, sums) + before;

  const unsigned int lo = tile * S.tile, hi = S.n - lo < S.tile ? S.n : lo + S.tile;
  for (unsigned int i0 = lo; i0 < hi; i0 += GA_EG_ROUND) {
    unsigned int k[GA_EG_KEYS], o[GA_EG_KEYS], digit[GA_EG_KEYS], at[GA_EG_KEYS];
    int live[GA_EG_KEYS];
#pragma unroll
    for (int j = 0; j < GA_EG_KEYS; j++) {
      const unsigned int i = i0 + (warp * GA_EG_KEYS + j) * 32 + lane;
      k[j] = o[j] = 0;
      live[j] = i < hi;
      if (live[j]) {
        k[j] = ga__eg_key_of(L, S, ids, key_in, i, nullptr);
        o[j] = S.pass == 0 ? i : order_in[i];
      }
      digit[j] = (k[j] >> shift) & (GA_EG_DIGITS - 1);
    }
    ga__eg_places(digit, live, base, cnt, at);
#pragma unroll
    for (int j = 0; j < GA_EG_KEYS; j++) {
      if (!live[j]) continue;
      key[at[j]] = k[j];
      if (S.pass + 1 == S.passes) off[at[j]] = ga__lm_offset<GA_EM_ND>(o[j], L.dims, L.t_str);
      else order[at[j]] = o[j];
    }
    __syncthreads();
  }
}

/* All passes in one launch, for as many tokens as the shared memory of a CTA or of one cluster
 * holds: CTA r of the cluster has the tokens, then the sorted keys, from r * GA_EG_TILE on. A pass counts
 * its digits, gives the counts to all CTAs, and sends every key to its place. */
#define GA_EG_TILE (GA_EG_ROUND * GA_EG_ROUNDS)
struct ga__eg_shared {
  ga__eg_table cnt;
  unsigned int tab[GA_EG_CLUSTER][GA_EG_DIGITS];
  unsigned int hist[GA_EG_DIGITS];
  unsigned int sums[GA_EG_WARPS];
  unsigned long long keys[GA_EG_TILE]; /* key << 32 | token */
};

/* all CTAs of the sort meet */
static __device__ __forceinline__ void ga__eg_meet() {
#if GA_EG_CLUSTER > 1
  ga__cluster_arrive();
  ga__cluster_wait();
#else
  __syncthreads();
#endif
}
template <typename T>
static __device__ __forceinline__ void ga__eg_put(T *p, unsigned int rank, T v) {
#if GA_EG_CLUSTER > 1
  ga__cluster_put(p, rank, v);
#else
  *p = v;
#endif
}

extern "C" __global__ void __launch_bounds__(GA_EG_THREADS)
#if GA_EG_CLUSTER > 1
    __cluster_dims__(GA_EG_CLUSTER, 1, 1)
#endif
ga_eg_sort_all(const __grid_constant__ ga__em_layout L, const __grid_constant__ ga__eg_sort S,
               const char *ids, unsigned int *key, long long *off, int *err) {
  ga__grid_dependency_sync();
  GA_LM_SHARED_DYNAMIC(ga__eg_shared, sh);
#if GA_EG_CLUSTER > 1
  ga__cluster_arrive(); /* waited for before the first store to another CTA's shared memory */
#endif
  const unsigned int d = threadIdx.x, lane = d % 32, warp = d / 32, r = blockIdx.x;
  unsigned int k[GA_EG_ROUNDS][GA_EG_KEYS], o[GA_EG_ROUNDS][GA_EG_KEYS];
#pragma unroll
  for (int g = 0; g < GA_EG_ROUNDS; g++)
#pragma unroll
    for (int j = 0; j < GA_EG_KEYS; j++) {
      const unsigned int i = r * GA_EG_TILE + g * GA_EG_ROUND + (warp * GA_EG_KEYS + j) * 32 + lane;
      o[g][j] = i;
      k[g][j] = i < S.n ? ga__eg_key(L, ids, i, err) : 0;
    }
#if GA_EG_CLUSTER > 1
  ga__cluster_wait();
#endif
  for (unsigned int pass = 0; pass < S.passes; pass++) {
    const unsigned int shift = pass * GA_EG_BITS;
    sh.hist[d] = 0;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < GA_EG_ROUNDS; g++)
#pragma unroll
      for (int j = 0; j < GA_EG_KEYS; j++)
        if (r * GA_EG_TILE + g * GA_EG_ROUND + (warp * GA_EG_KEYS + j) * 32 + lane < S.n)
          atomicAdd(&sh.hist[(k[g][j] >> shift) & (GA_EG_DIGITS - 1)], 1u);
    __syncthreads();
    for (unsigned int t = 0; t < GA_EG_CLUSTER; t++) ga__eg_put(&sh.tab[r][d], t, sh.hist[d]);
    /* behind this everybody has the counts, and has taken its keys out of `keys` */
    ga__eg_meet();
    unsigned int total = 0, before = 0;
#pragma unroll
    for (unsigned int t = 0; t < GA_EG_CLUSTER; t++) {
      const unsigned int x = sh.tab[t][d];
      total += x;
      before += t < r ? x : 0;
    }
    unsigned int base = ga__eg_prefix(total, sh.sums) + before;
#pragma unroll
    for (int g = 0; g < GA_EG_ROUNDS; g++) {
      unsigned int digit[GA_EG_KEYS], at[GA_EG_KEYS];
      int live[GA_EG_KEYS];
#pragma unroll
      for (int j = 0; j < GA_EG_KEYS; j++) {
        live[j] = r * GA_EG_TILE + g * GA_EG_ROUND + (warp * GA_EG_KEYS + j) * 32 + lane < S.n;
        digit[j] = (k[g][j] >> shift) & (GA_EG_DIGITS - 1);
      }
      ga__eg_places(digit, live, base, sh.cnt, at);
#pragma unroll
      for (int j = 0; j < GA_EG_KEYS; j++) {
        if (!live[j]) continue;
        if (GA_EG_CLUSTER > 1 && pass + 1 == S.passes) {
          key[at[j]] = k[g][j];
          off[at[j]] = ga__lm_offset<GA_EM_ND>(o[g][j], L.dims, L.t_str);
        } else {
          ga__eg_put(&sh.keys[at[j] % GA_EG_TILE], at[j] / GA_EG_TILE,
                     (unsigned long long)k[g][j] << 32 | o[g][j]);
        }
      }
      __syncthreads();
    }
    if (GA_EG_CLUSTER > 1 && pass + 1 == S.passes) return;
    ga__eg_meet(); /* every key has arrived */
    if (pass + 1 == S.passes) break;
#pragma unroll
    for (int g = 0; g < GA_EG_ROUNDS; g++)
#pragma unroll
      for (int j = 0; j < GA_EG_KEYS; j++) {
        const unsigned long long x = sh.keys[g * GA_EG_ROUND + (warp * GA_EG_KEYS + j) * 32 + lane];
        k[g][j] = (unsigned int)(x >> 32);
        o[g][j] = (unsigned int)x;
      }
  }
  /* One CTA's lists leave in order: its scattered stores would take a cycle for each key (4096
   * tokens 15.6 us, so 12.5). A cluster's have as many SMs to leave from. */
  for (unsigned int i = d; i < GA_EG_TILE && r * GA_EG_TILE + i < S.n; i += GA_EG_THREADS) {
    const unsigned long long x = sh.keys[i];
    key[r * GA_EG_TILE + i] = (unsigned int)(x >> 32);
    off[r * GA_EG_TILE + i] = ga__lm_offset<GA_EM_ND>((unsigned int)x, L.dims, L.t_str);
  }
}

/* ---- summing ---- */
/* tokens whose rows a thread has in flight, 16 bytes of each, in 4 CTAs an SM. Twice as many in half
 * as many CTAs are as many bytes, but fewer warps to go on while a run's end is written; rows moved
 * in several narrow vectors take more registers (two parts of 8190 rows of 1021 floats: 100 us with
 * 2, 107 with 4, 125 with 4 in 2 CTAs; 32760 rows of 2048 halfs: 126 with 2, 119 with 4). */
#define GA_EG_U (GA_EM_C > 1 ? 2 : 4)
#define GA_EG_J 4 /* parts a thread has in flight */

static __device__ __forceinline__ void ga__eg_park(GA_EM_F_T *p, const GA_EM_F_T acc[GA_EM_N]) {
#pragma unroll
  for (int j = 0; j < GA_EM_N; j++) p[j] = acc[j];
}

/* Sums sorted tokens [lo, hi) of n at a thread's vectors; off: their rows of dout. head, tail:
 * where the parts of the run that began before lo, and of the one that goes on behind hi, are
 * parked. Both lists may be read up to GA_EG_U - 1 entries beyond hi, by vectors where WIDE (lo a
 * multiple of GA_EG_U). */
template <int WIDE>
static __device__ __forceinline__ void ga__eg_chunk(const ga__em_layout &L, char *dtable,
                                                    const char *dout, const unsigned int *key,
                                                    const long long *off, unsigned int n,
                                                    unsigned int lo, unsigned int hi, ga__em_pos pos,
                                                    GA_EM_F_T *head, GA_EM_F_T *tail) {
  const unsigned int none = (unsigned int)L.v;
  unsigned int cur = key[lo];
  int open_head = lo > 0 && key[lo - 1] == cur;
  GA_EM_F_T acc[GA_EM_N];
#pragma unroll
  for (int j = 0; j < GA_EM_N; j++) acc[j] = 0;
  ga__em_out old; /* of row `cur` */
  for (unsigned int i = lo; i < hi && cur != none; i += GA_EG_U) {
    struct alignas(4 * GA_EG_U) { /* i is a multiple of GA_EG_U */
      unsigned int v[GA_EG_U];
    } k;
    struct alignas(16) {
      long long v[GA_EG_U];
    } at;
    ga__em_in q[GA_EG_U];
#if GA_EM_ACCUMULATE
    ga__em_out held[GA_EG_U]; /* the rows that the tokens' runs are added to */
#endif
    if (WIDE) {
      k = *reinterpret_cast<const decltype(k) *>(key + i);
      at = *reinterpret_cast<const decltype(at) *>(off + i);
    } else {
#pragma unroll
      for (int u = 0; u < GA_EG_U; u++) {
        k.v[u] = key[i + u];
        at.v[u] = off[i + u];
      }
    }
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++) {
      if (i + u >= hi) k.v[u] = none;
      if (k.v[u] != none)
        q[u] = ga__em_read<ga__em_in, ga__em_in1>(dout + at.v[u], L.t_col, pos);
    }
#if GA_EM_ACCUMULATE
    /* read with the tokens' rows, not when a run ends: once a run, at its first token here */
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++)
      if (k.v[u] != none && (u == 0 ? k.v[u] != cur || i == lo : k.v[u] != k.v[u - 1]))
        held[u] = ga__eg_held(L, dtable, k.v[u], pos);
    if (i == lo) old = held[0];
#endif
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++) {
      if (i + u >= hi) break;
      if (k.v[u] != cur) { /* the run ends inside the chunk */
        if (open_head) ga__eg_park(head, acc);
        else ga__eg_write(L, dtable, cur, pos, acc, old);
        open_head = 0;
        cur = k.v[u];
#if GA_EM_ACCUMULATE
        old = held[u];
#endif
#pragma unroll
        for (int j = 0; j < GA_EM_N; j++) acc[j] = 0;
        if (cur == none) break;
      }
      GA_EM_F_T x[GA_EM_N];
      ga__em_get<GA_EM_A_T>(x, q[u]);
#pragma unroll
      for (int j = 0; j < GA_EM_N; j++) acc[j] += x[j];
    }
  }
  if (cur == none) return;
  if (open_head) ga__eg_park(head, acc);
  else if (hi < n && key[hi] == cur) ga__eg_park(tail, acc);
  else ga__eg_write(L, dtable, cur, pos, acc, old);
}

/* Joins the run that starts in chunk c (tokens c * size ...) and goes on in the next, if there is
 * one: of the `ny` threads at a vector position thread y takes every ny-th part, then the first
 * adds their sums, always in the same order; with ny > 1 all threads of a warp, or of the CTA where
 * there are 32 or more along the row, are here for the same c. part: the chunks' parked rows at this thread's vectors, heads and tails in turn, `step`
 * elements apart. sum: with ny > 1, 256 * GA_EM_N entries of shared memory. */
static __device__ __forceinline__ void ga__eg_join_run(const ga__em_layout &L, char *dtable,
                                                       const unsigned int *key, unsigned int c,
                                                       unsigned int size, unsigned int chunks,
                                                       ga__em_pos pos, const GA_EM_F_T *part,
                                                       size_t step, unsigned int y, unsigned int ny,
                                                       GA_EM_F_T *sum) {
  const unsigned int lo = c * size, next = lo + size; /* next < n: chunk c + 1 exists */
  const unsigned int cur = key[next];
  if (cur == (unsigned int)L.v || key[next - 1] != cur) return;
  if (key[lo] == cur && lo > 0 && key[lo - 1] == cur) return; /* it began earlier */
  const int inside = pos.v < L.nv;
  GA_EM_F_T acc[GA_EM_N];
  ga__em_out old;
  if (inside) {
#pragma unroll
    for (int j = 0; j < GA_EM_N; j++) acc[j] = 0;
    if (y == 0) {
#if GA_EM_ACCUMULATE
      old = ga__eg_held(L, dtable, cur, pos);
#endif
      const GA_EM_F_T *p = part + (2 * (size_t)c + 1) * step;
#pragma unroll
      for (int j = 0; j < GA_EM_N; j++) acc[j] = p[j];
    }
    /* GA_EG_J parts are fetched together with the keys that tell whether they belong to the run */
    for (unsigned int d = c + 1 + y, more = 1; more && d < chunks; d += GA_EG_J * ny) {
      GA_EM_F_T x[GA_EG_J][GA_EM_N];
      unsigned int k[GA_EG_J];
#pragma unroll
      for (int u = 0; u < GA_EG_J; u++)
        if (d + u * ny < chunks) {
          k[u] = key[(d + u * ny) * size];
          const GA_EM_F_T *p = part + 2 * (size_t)(d + u * ny) * step;
#pragma unroll
          for (int j = 0; j < GA_EM_N; j++) x[u][j] = p[j];
        }
#pragma unroll
      for (int u = 0; u < GA_EG_J; u++) {
        if (!more || d + u * ny >= chunks || k[u] != cur) {
          more = 0;
          continue;
        }
#pragma unroll
        for (int j = 0; j < GA_EM_N; j++) acc[j] += x[u][j];
      }
    }
    if (y > 0) ga__eg_park(sum + (threadIdx.y * blockDim.x + threadIdx.x) * GA_EM_N, acc);
  }
  if (ny > 1) {
    if (blockDim.x < 32) __syncwarp();
    else __syncthreads();
  }
  if (!inside || y > 0) return;
  for (unsigned int i = 1; i < ny; i++)
#pragma unroll
    for (int j = 0; j < GA_EM_N; j++) acc[j] += sum[((threadIdx.y + i) * blockDim.x + threadIdx.x) * GA_EM_N + j];
  ga__eg_write(L, dtable, cur, pos, acc, old);
}

/* `part` holds GA_EM_N sums for each thread along the row, two rows of them per chunk. */
extern "C" __global__ void __launch_bounds__(256, 4)
ga_eg_sum(const __grid_constant__ ga__em_layout L, char *dtable, const char *dout,
          const unsigned int *key, const long long *off, GA_EM_F_T *part) {
  ga__grid_dependency_sync();
  const ga__em_pos pos = ga__em_here(L);
  const unsigned int c = blockIdx.x * blockDim.y + threadIdx.y;
  if (pos.v >= L.nv || c >= L.chunks) return;
  const unsigned int n = (unsigned int)L.n, lo = c * L.chunk, hi = n - lo < L.chunk ? n : lo + L.chunk;
  const size_t step = (size_t)gridDim.y * blockDim.x * GA_EM_N;
  GA_EM_F_T *head = part + 2 * (size_t)c * step + (size_t)(blockIdx.y * blockDim.x + threadIdx.x) * GA_EM_N;
  ga__eg_chunk<1>(L, dtable, dout, key, off, n, lo, hi, pos, head, head + step);
}

/* A CTA for each chunk but the last (blockIdx.x) and slice of the rows, with as many threads along
 * them as in ga_eg_sum; a warp where these are fewer than 32. Most find nothing to join. */
extern "C" __global__ void __launch_bounds__(256)
ga_eg_join(const __grid_constant__ ga__em_layout L, char *dtable, const unsigned int *key,
           const GA_EM_F_T *part) {
  ga__grid_dependency_sync();
  __shared__ GA_EM_F_T sum[256 * GA_EM_N];
  const unsigned int narrow = blockDim.x < 32, ny = narrow ? 32 / blockDim.x : blockDim.y;
  const unsigned int c = narrow ? blockIdx.x * 8 + threadIdx.y / ny : blockIdx.x;
  if (c + 1 >= L.chunks) return; /* whole warps */
  ga__eg_join_run(L, dtable, key, c, L.chunk, L.chunks, ga__em_here(L),
                  part + (size_t)(blockIdx.y * blockDim.x + threadIdx.x) * GA_EM_N,
                  (size_t)gridDim.y * blockDim.x * GA_EM_N, threadIdx.y % ny, ny, sum);
}

/* ---- few tokens ---- */
#define GA_EG_FEW 1024 /* tokens at most */
#define GA_EG_FEW_WARPS 8
#define GA_EG_TX 32   /* vector positions of a CTA at most; blockDim.x * blockDim.y is 256 */

/* CTA (x, y) owns L.chunk rows from x * L.chunk and slice y of their vectors. */
extern "C" __global__ void __launch_bounds__(256)
ga_eg_direct(const __grid_constant__ ga__em_layout L, char *dtable, const char *dout,
             const char *ids, int *err) {
  ga__grid_dependency_sync();
  __shared__ unsigned int key[GA_EG_FEW + GA_EG_U], found[GA_EG_FEW_WARPS];
  __shared__ long long off[GA_EG_FEW + GA_EG_U];
  /* the rows and numbers of the CTA's tokens; when these are sorted, the parts of runs */
  alignas(16) __shared__ char both[sizeof(GA_EM_F_T) * 256 * 2 * GA_EM_N > 8 * GA_EG_FEW
                                       ? sizeof(GA_EM_F_T) * 256 * 2 * GA_EM_N : 8 * GA_EG_FEW];
  unsigned int *row = reinterpret_cast<unsigned int *>(both), *token = row + GA_EG_FEW;
  GA_EM_F_T *part = reinterpret_cast<GA_EM_F_T *>(both);
  const unsigned int tid = threadIdx.y * blockDim.x + threadIdx.x, lane = tid % 32, warp = tid / 32;
  const unsigned int n = (unsigned int)L.n;
  const unsigned long long r0 = (unsigned long long)blockIdx.x * L.chunk;
  const unsigned long long r1 = L.v - r0 < L.chunk ? L.v : r0 + L.chunk;
  /* all keys are on their way, and the zeros, before the first is looked at (1024 halfs on (32000,
   * 1024): 18.5 us; keys 256 at a time with zeros after the sort: 19.8; 20 tokens: 4.0 and 3.9) */
  unsigned int all_keys[GA_EG_FEW / 256];
#pragma unroll
  for (int j = 0; j < GA_EG_FEW / 256; j++) {
    const unsigned int i = j * 256 + tid;
    all_keys[j] = i < n ? ga__eg_key(L, ids, i, blockIdx.x == 0 && blockIdx.y == 0 ? err : nullptr) : (unsigned int)L.v;
  }
  const ga__em_pos pos = ga__em_here(L);
#if !GA_EM_ACCUMULATE
  if (pos.v < L.nv)
    for (unsigned long long r = r0 + threadIdx.y; r < r1; r += blockDim.y)
      ga__em_write(dtable + (long long)r * L.v_row, L.v_col, pos, ga__em_zero<ga__em_out>());
#endif
  /* the tokens of these rows, in their order */
  unsigned int m = 0;
#pragma unroll
  for (int j = 0; j < GA_EG_FEW / 256; j++) {
    if (j * 256 >= n) break;
    const unsigned int r = all_keys[j];
    const int mine = r >= r0 && r < r1;
    const unsigned int all = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) found[warp] = __popc(all);
    __syncthreads();
    unsigned int at = m + __popc(all & ((1u << lane) - 1));
    for (unsigned int w = 0; w < GA_EG_FEW_WARPS; w++) {
      at += w < warp ? found[w] : 0;
      m += found[w];
    }
    if (mine) {
      row[at] = r;
      token[at] = j * 256 + tid;
    }
    __syncthreads();
  }
  /* sorted by row: a token's place is the number of those before it */
  for (unsigned int i = tid; i < m; i += 256) {
    const unsigned int k = row[i];
    unsigned int at = 0;
    if (r1 - r0 == 1) at = i; /* one row: in order already */
    else
#pragma unroll 4
      for (unsigned int j = 0; j < m; j++) at += row[j] < k + (j < i);
    key[at] = k;
    off[at] = ga__lm_offset<GA_EM_ND>(token[i], L.dims, L.t_str);
  }
  __syncthreads();
  if (m == 0) return;
  const unsigned int size = (m + blockDim.y - 1) / blockDim.y, chunks = (m + size - 1) / size;
  const unsigned int c = threadIdx.y;
  GA_EM_F_T *mine = part + threadIdx.x * GA_EM_N;
  const size_t step = (size_t)blockDim.x * GA_EM_N;
  if (pos.v < L.nv && c < chunks)
    ga__eg_chunk<0>(L, dtable, dout, key, off, m, c * size, m - c * size < size ? m : (c + 1) * size, pos,
                 mine + 2 * c * step, mine + (2 * c + 1) * step);
  __syncthreads();
  if (pos.v < L.nv && c + 1 < chunks) ga__eg_join_run(L, dtable, key, c, size, chunks, pos, mine, step, 0, 1, mine);
}
#endif
