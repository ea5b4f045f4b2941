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

typedef ga__lm_vec<GA_EM_A_T, GA_EM_E> ga__em_in;
typedef ga__lm_vec<GA_EM_O_T, GA_EM_E> ga__em_out;

#ifdef GA_EM_BUILD_LOOKUP
#define GA_EM_U 8        /* loads of a thread in flight */
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
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
  if (v >= L.nv) return;
  const GA_EM_F_T scale = (GA_EM_F_T)L.scale;
  const char *col = table + (long long)v * GA_EM_E * L.v_col;
  char *dst = out + (long long)v * GA_EM_E * L.t_col;
  const unsigned int t1 = (threadIdx.y + 1) * L.chunk;
  for (unsigned int t = threadIdx.y * L.chunk; t < t1; t += GA_EM_U) {
    ga__em_in q[GA_EM_U];
#pragma unroll
    for (int u = 0; u < GA_EM_U; u++) {
#pragma unroll
      for (int j = 0; j < (int)(sizeof(q[u].w) / sizeof(q[u].w[0])); j++) q[u].w[j] = 0;
      if (t + u < t1 && to[t + u] != GA_EM_NOWHERE && from[t + u] != GA_EM_NOWHERE)
        q[u] = ga__lm_load<ga__em_in>(col + from[t + u]);
    }
#pragma unroll
    for (int u = 0; u < GA_EM_U; u++) {
      if (t + u >= t1 || to[t + u] == GA_EM_NOWHERE) continue;
      GA_EM_F_T x[GA_EM_E];
      ga__lm_get<GA_EM_A_T, GA_EM_E>(x, q[u]);
#pragma unroll
      for (int j = 0; j < GA_EM_E; j++) x[j] *= scale;
      ga__em_out o;
      ga__lm_put<GA_EM_O_T, GA_EM_E>(o, x);
      ga__lm_store(dst + to[t + u], o);
    }
  }
}
#endif

#ifdef GA_EM_BUILD_GRAD
/* The gradient is a sum over SORTED tokens, in launches that depend on nothing
 * but the ids' values, so that the result is the same bits every time.
 *
 * Few tokens: ga_eg_direct. A CTA owns a range of table rows and a slice of
 * their vectors, picks its tokens from all ids, sorts them in shared memory,
 * writes zeros and sums.
 *
 * Many tokens: the tokens are sorted by row and, within a row, by token (a
 * radix sort of GA_EG_BITS bits a pass: ga_eg_count, then ga_eg_scatter for
 * each pass, which also counts for the next). Tokens that contribute nothing
 * get the key V and go last. The CTAs beyond the sort's write the zeros of the
 * rows, a part of them in each launch, so that the sort hides behind them.
 * Then ga_eg_sum: the sorted tokens are cut into equal chunks; a group of
 * threads sums a chunk's rows, one vector position per thread. A run of equal
 * keys that lies inside the chunk is finished and written; the parts of runs
 * that cross a chunk's ends are parked, two rows per chunk. ga_eg_join: the
 * group of the chunk in which a crossing run starts adds its parts in order
 * and writes the row. */

/* zeros for a part of dtable: flat bytes where its rows are adjacent, else row by row */
struct ga__eg_fill {
  char *p;
  unsigned long long bytes; /* > 0: flat */
  unsigned long long r0, r1; /* rows, otherwise */
};

static __device__ __forceinline__ char *ga__eg_place(const ga__em_layout &L, char *dtable,
                                                     unsigned int row, unsigned int v) {
  return dtable + (long long)row * L.v_row + (long long)v * GA_EM_E * L.v_col;
}

/* `old`: what the row holds so far, read ahead by the caller (used where it is added to) */
static __device__ __forceinline__ void ga__eg_write(const ga__em_layout &L, char *dtable,
                                                    unsigned int row, unsigned int v,
                                                    const GA_EM_F_T acc[GA_EM_E],
                                                    const ga__em_out &old) {
  const GA_EM_F_T scale = (GA_EM_F_T)L.scale;
  char *p = ga__eg_place(L, dtable, row, v);
  GA_EM_F_T x[GA_EM_E];
  ga__em_out q;
#if GA_EM_ACCUMULATE
  ga__lm_get<GA_EM_O_T, GA_EM_E>(x, old);
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) x[j] += acc[j] * scale;
#else
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) x[j] = acc[j] * scale;
#endif
  ga__lm_put<GA_EM_O_T, GA_EM_E>(q, x);
  ga__lm_store(p, q);
}

static __device__ __forceinline__ void ga__eg_zero_row(const ga__em_layout &L, char *dtable,
                                                       unsigned long long row, unsigned int v) {
  ga__em_out q;
#pragma unroll
  for (int j = 0; j < (int)(sizeof(q.w) / sizeof(q.w[0])); j++) q.w[j] = 0;
  ga__lm_store(dtable + (long long)row * L.v_row + (long long)v * GA_EM_E * L.v_col, q);
}

static __device__ __forceinline__ void ga__eg_zeros(const ga__em_layout &L, const ga__eg_fill &F,
                                                    unsigned int cta, unsigned int ctas) {
  if (F.bytes > 0) {
    const unsigned long long n = F.bytes / 16, step = (unsigned long long)ctas * blockDim.x;
    ga__lm_raw<16> q;
    q.w[0] = q.w[1] = q.w[2] = q.w[3] = 0;
    for (unsigned long long i = (unsigned long long)cta * blockDim.x + threadIdx.x; i < n; i += step)
      ga__lm_store(F.p + i * 16, q);
    /* what is left is less than 16 bytes */
    if (cta == 0 && threadIdx.x < F.bytes - n * 16) F.p[n * 16 + threadIdx.x] = 0;
    return;
  }
  const unsigned int lane = threadIdx.x % 32, warps = blockDim.x / 32;
  for (unsigned long long r = F.r0 + (unsigned long long)cta * warps + threadIdx.x / 32; r < F.r1;
       r += (unsigned long long)ctas * warps)
    for (unsigned int v = lane; v < L.nv; v += 32) ga__eg_zero_row(L, F.p, r, v);
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

/* counts[pass][digit][tile]: how many keys of a tile have the digit. The first pass's are counted
 * here, the others' are set to zero for ga_eg_scatter to add to. */
extern "C" __global__ void __launch_bounds__(GA_EG_THREADS)
ga_eg_count(const __grid_constant__ ga__em_layout L, const __grid_constant__ ga__eg_sort S,
            const __grid_constant__ ga__eg_fill F, unsigned int *counts, const char *ids, int *err) {
  ga__grid_dependency_sync();
  if (blockIdx.x >= S.tiles) {
    ga__eg_zeros(L, F, blockIdx.x - S.tiles, gridDim.x - S.tiles);
    return;
  }
  __shared__ unsigned int hist[GA_EG_DIGITS];
  const unsigned int d = threadIdx.x, tile = blockIdx.x;
  hist[d] = 0;
  __syncthreads();
  const unsigned int lo = tile * S.tile, hi = S.n - lo < S.tile ? S.n : lo + S.tile;
  for (unsigned int i = lo + threadIdx.x; i < hi; i += GA_EG_THREADS)
    atomicAdd(&hist[ga__eg_key(L, ids, i, err) & (GA_EG_DIGITS - 1)], 1u);
  __syncthreads();
  counts[d * S.tiles + tile] = hist[d];
  for (unsigned int p = 1; p < S.passes; p++)
    counts[(p * GA_EG_DIGITS + d) * S.tiles + tile] = 0;
}

/* One pass: every key goes behind all with a smaller digit and, with an equal digit, behind those
 * that stand before it. The first pass takes the ids themselves; the last one leaves the byte
 * offsets of the tokens' rows of dout, so that the sums need no division. */
extern "C" __global__ void __launch_bounds__(GA_EG_THREADS)
ga_eg_scatter(const __grid_constant__ ga__em_layout L, const __grid_constant__ ga__eg_sort S,
              const __grid_constant__ ga__eg_fill F, unsigned int *counts, const char *ids,
              const unsigned int *key_in, const unsigned int *order_in, unsigned int *key,
              unsigned int *order, long long *off) {
  ga__grid_dependency_sync();
  if (blockIdx.x >= S.tiles) {
    ga__eg_zeros(L, F, blockIdx.x - S.tiles, gridDim.x - S.tiles);
    return;
  }
  __shared__ unsigned int cnt[GA_EG_WARPS][GA_EG_DIGITS];
  __shared__ unsigned int sums[GA_EG_WARPS];
  const unsigned int d = threadIdx.x, lane = d % 32, warp = d / 32, tile = blockIdx.x;
  const unsigned int shift = S.pass * GA_EG_BITS;

  /* where the digit's keys of this tile begin */
  const unsigned int *c = counts + (S.pass * GA_EG_DIGITS + d) * S.tiles;
  unsigned int total = 0, before = 0;
  for (unsigned int t = 0; t < S.tiles; t++) {
    const unsigned int x = c[t];
    total += x;
    before += t < tile ? x : 0;
  }
  unsigned int scan = total;
#pragma unroll
  for (int s = 1; s < 32; s *= 2) {
    const unsigned int o = __shfl_up_sync(0xffffffffu, scan, s);
    if (lane >= (unsigned int)s) scan += o;
  }
  if (lane == 31) sums[warp] = scan;
  __syncthreads();
  unsigned int base = scan - total + before;
  for (unsigned int w = 0; w < warp; w++) base += sums[w];

  const unsigned int lo = tile * S.tile, hi = S.n - lo < S.tile ? S.n : lo + S.tile;
  for (unsigned int i0 = lo; i0 < hi; i0 += GA_EG_ROUND) {
    unsigned int k[GA_EG_KEYS], o[GA_EG_KEYS], rank[GA_EG_KEYS];
#pragma unroll
    for (int j = 0; j < GA_EG_KEYS; j++) { /* a warp's keys are adjacent */
      const unsigned int i = i0 + (warp * GA_EG_KEYS + j) * 32 + lane;
      k[j] = o[j] = 0;
      if (i < hi) {
        k[j] = S.pass == 0 ? ga__eg_key(L, ids, i, nullptr) : key_in[i];
        o[j] = S.pass == 0 ? i : order_in[i];
      }
    }
    for (int w = 0; w < GA_EG_WARPS; w++) cnt[w][d] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < GA_EG_KEYS; j++) {
      const unsigned int i = i0 + (warp * GA_EG_KEYS + j) * 32 + lane;
      const unsigned int digit = i < hi ? (k[j] >> shift) & (GA_EG_DIGITS - 1) : GA_EG_DIGITS;
      const unsigned int same = __match_any_sync(0xffffffffu, digit);
      const unsigned int seen = i < hi ? cnt[warp][digit] : 0;
      rank[j] = seen + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (i < hi && __ffs(same) - 1 == (int)lane) cnt[warp][digit] = seen + __popc(same);
      __syncwarp();
    }
    __syncthreads();
    for (int w = 0; w < GA_EG_WARPS; w++) { /* the digit's place for each warp */
      const unsigned int x = cnt[w][d];
      cnt[w][d] = base;
      base += x;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < GA_EG_KEYS; j++) {
      const unsigned int i = i0 + (warp * GA_EG_KEYS + j) * 32 + lane;
      if (i < hi) {
        const unsigned int at = cnt[warp][(k[j] >> shift) & (GA_EG_DIGITS - 1)] + rank[j];
        key[at] = k[j];
        if (S.pass + 1 == S.passes) {
          off[at] = ga__lm_offset<GA_EM_ND>(o[j], L.dims, L.t_str);
        } else {
          order[at] = o[j];
          atomicAdd(&counts[((S.pass + 1) * GA_EG_DIGITS + ((k[j] >> (shift + GA_EG_BITS)) & (GA_EG_DIGITS - 1))) * S.tiles + at / S.tile], 1u);
        }
      }
    }
    __syncthreads();
  }
}

/* ---- summing ---- */
#define GA_EG_U 8
#define GA_EG_J 8

static __device__ __forceinline__ void ga__eg_park(GA_EM_F_T *p, const GA_EM_F_T acc[GA_EM_E]) {
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) p[j] = acc[j];
}

/* Sums sorted tokens [lo, hi) of n at vector position v; off: their rows of dout. head, tail:
 * where the parts of the run that began before lo, and of the one that goes on behind hi, are
 * parked. Both lists may be read up to GA_EG_U - 1 entries beyond hi, by vectors where WIDE (lo a
 * multiple of GA_EG_U). */
template <int WIDE>
static __device__ __forceinline__ void ga__eg_chunk(const ga__em_layout &L, char *dtable,
                                                    const char *dout, const unsigned int *key,
                                                    const long long *off, unsigned int n,
                                                    unsigned int lo, unsigned int hi, unsigned int v,
                                                    GA_EM_F_T *head, GA_EM_F_T *tail) {
  const unsigned int none = (unsigned int)L.v;
  unsigned int cur = key[lo];
  int open_head = lo > 0 && key[lo - 1] == cur;
  GA_EM_F_T acc[GA_EM_E];
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) acc[j] = 0;
  ga__em_out old; /* of row `cur` */
  const char *col = dout + (long long)v * GA_EM_E * L.t_col;
  for (unsigned int i = lo; i < hi && cur != none; i += GA_EG_U) {
    struct alignas(16) {
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
        q[u] = ga__lm_load<ga__em_in>(col + at.v[u]);
    }
#if GA_EM_ACCUMULATE
    /* read with the tokens' rows, not when a run ends: once a run, at its first token here */
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++)
      if (k.v[u] != none && (u == 0 ? k.v[u] != cur || i == lo : k.v[u] != k.v[u - 1]))
        held[u] = ga__lm_load<ga__em_out>(ga__eg_place(L, dtable, k.v[u], v));
    if (i == lo) old = held[0];
#endif
#pragma unroll
    for (int u = 0; u < GA_EG_U; u++) {
      if (i + u >= hi) break;
      if (k.v[u] != cur) { /* the run ends inside the chunk */
        if (open_head) ga__eg_park(head, acc);
        else ga__eg_write(L, dtable, cur, v, acc, old);
        open_head = 0;
        cur = k.v[u];
#if GA_EM_ACCUMULATE
        old = held[u];
#endif
#pragma unroll
        for (int j = 0; j < GA_EM_E; j++) acc[j] = 0;
        if (cur == none) break;
      }
      GA_EM_F_T x[GA_EM_E];
      ga__lm_get<GA_EM_A_T, GA_EM_E>(x, q[u]);
#pragma unroll
      for (int j = 0; j < GA_EM_E; j++) acc[j] += x[j];
    }
  }
  if (cur == none) return;
  if (open_head) ga__eg_park(head, acc);
  else if (hi < n && key[hi] == cur) ga__eg_park(tail, acc);
  else ga__eg_write(L, dtable, cur, v, acc, old);
}

/* Joins the run that starts in chunk c (tokens c * size ...) and goes on in the next, if there is
 * one. part: the chunks' parked rows at this vector position, heads and tails in turn, `step`
 * elements apart. */
static __device__ __forceinline__ void ga__eg_join_run(const ga__em_layout &L, char *dtable,
                                                       const unsigned int *key, unsigned int c,
                                                       unsigned int size, unsigned int chunks,
                                                       unsigned int v, const GA_EM_F_T *part,
                                                       size_t step) {
  const unsigned int lo = c * size, next = lo + size; /* next < n: chunk c + 1 exists */
  const unsigned int cur = key[next];
  if (cur == (unsigned int)L.v || key[next - 1] != cur) return;
  if (key[lo] == cur && lo > 0 && key[lo - 1] == cur) return; /* it began earlier */
  GA_EM_F_T acc[GA_EM_E];
  const GA_EM_F_T *p = part + (2 * (size_t)c + 1) * step;
#pragma unroll
  for (int j = 0; j < GA_EM_E; j++) acc[j] = p[j];
  ga__em_out old;
#if GA_EM_ACCUMULATE
  old = ga__lm_load<ga__em_out>(ga__eg_place(L, dtable, cur, v));
#endif
  /* GA_EG_J parts are fetched together with the keys that tell whether they belong to the run */
  for (unsigned int d = c + 1, more = 1; more && d < chunks; d += GA_EG_J) {
    GA_EM_F_T x[GA_EG_J][GA_EM_E];
    unsigned int k[GA_EG_J];
#pragma unroll
    for (int u = 0; u < GA_EG_J; u++)
      if (d + u < chunks) {
        k[u] = key[(d + u) * size];
        p = part + 2 * (size_t)(d + u) * step;
#pragma unroll
        for (int j = 0; j < GA_EM_E; j++) x[u][j] = p[j];
      }
#pragma unroll
    for (int u = 0; u < GA_EG_J; u++) {
      if (!more || d + u >= chunks || k[u] != cur) {
        more = 0;
        continue;
      }
#pragma unroll
      for (int j = 0; j < GA_EM_E; j++) acc[j] += x[u][j];
    }
  }
  ga__eg_write(L, dtable, cur, v, acc, old);
}

extern "C" __global__ void __launch_bounds__(256)
ga_eg_sum(const __grid_constant__ ga__em_layout L, char *dtable, const char *dout,
          const unsigned int *key, const long long *off, GA_EM_F_T *part) {
  ga__grid_dependency_sync();
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
  const unsigned int c = blockIdx.x * blockDim.y + threadIdx.y;
  if (v >= L.nv || c >= L.chunks) return;
  const unsigned int n = (unsigned int)L.n, lo = c * L.chunk, hi = n - lo < L.chunk ? n : lo + L.chunk;
  GA_EM_F_T *head = part + (2 * (size_t)c * L.nv + v) * GA_EM_E;
  ga__eg_chunk<1>(L, dtable, dout, key, off, n, lo, hi, v, head, head + (size_t)L.nv * GA_EM_E);
}

extern "C" __global__ void __launch_bounds__(256)
ga_eg_join(const __grid_constant__ ga__em_layout L, char *dtable, const unsigned int *key,
           const GA_EM_F_T *part) {
  ga__grid_dependency_sync();
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
  const unsigned int c = blockIdx.x * blockDim.y + threadIdx.y;
  if (v >= L.nv || c + 1 >= L.chunks) return;
  ga__eg_join_run(L, dtable, key, c, L.chunk, L.chunks, v, part + (size_t)v * GA_EM_E,
                  (size_t)L.nv * GA_EM_E);
}

/* ---- few tokens ---- */
#define GA_EG_FEW 512 /* tokens at most */
#define GA_EG_FEW_WARPS 8
#define GA_EG_TX 32   /* vector positions of a CTA at most; blockDim.x * blockDim.y is 256 */

/* CTA (x, y) owns L.chunk rows from x * L.chunk and the vectors of slice y. */
extern "C" __global__ void __launch_bounds__(256)
ga_eg_direct(const __grid_constant__ ga__em_layout L, char *dtable, const char *dout,
             const char *ids, int *err) {
  ga__grid_dependency_sync();
  __shared__ unsigned int row[GA_EG_FEW], token[GA_EG_FEW], key[GA_EG_FEW + GA_EG_U];
  __shared__ long long off[GA_EG_FEW + GA_EG_U];
  __shared__ unsigned int found[GA_EG_FEW_WARPS];
  __shared__ GA_EM_F_T part[256 * 2 * GA_EM_E];
  const unsigned int tid = threadIdx.y * blockDim.x + threadIdx.x, lane = tid % 32, warp = tid / 32;
  const unsigned int n = (unsigned int)L.n;
  const unsigned long long r0 = (unsigned long long)blockIdx.x * L.chunk;
  const unsigned long long r1 = L.v - r0 < L.chunk ? L.v : r0 + L.chunk;
  /* the tokens of these rows, in their order */
  unsigned int m = 0;
  for (unsigned int i0 = 0; i0 < n; i0 += 256) {
    const unsigned int i = i0 + tid;
    unsigned long long r = L.v;
    if (i < n) r = ga__eg_key(L, ids, i, blockIdx.x == 0 && blockIdx.y == 0 ? err : nullptr);
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
      row[at] = (unsigned int)r;
      token[at] = i;
    }
    __syncthreads();
  }
  /* sorted by row: a token's place is the number of those before it */
  for (unsigned int i = tid; i < m; i += 256) {
    const unsigned int k = row[i];
    unsigned int at = 0;
    for (unsigned int j = 0; j < m; j++) at += row[j] < k || (row[j] == k && j < i);
    key[at] = k;
    off[at] = ga__lm_offset<GA_EM_ND>(token[i], L.dims, L.t_str);
  }
  const unsigned int v = blockIdx.y * blockDim.x + threadIdx.x;
#if !GA_EM_ACCUMULATE
  if (v < L.nv)
    for (unsigned long long r = r0 + threadIdx.y; r < r1; r += blockDim.y) ga__eg_zero_row(L, dtable, r, v);
#endif
  __syncthreads();
  if (m == 0) return;
  const unsigned int size = (m + blockDim.y - 1) / blockDim.y, chunks = (m + size - 1) / size;
  const unsigned int c = threadIdx.y;
  GA_EM_F_T *mine = part + threadIdx.x * GA_EM_E;
  const size_t step = (size_t)blockDim.x * GA_EM_E;
  if (v < L.nv && c < chunks)
    ga__eg_chunk<0>(L, dtable, dout, key, off, m, c * size, m - c * size < size ? m : (c + 1) * size, v,
                 mine + 2 * c * step, mine + (2 * c + 1) * step);
  __syncthreads();
  if (v < L.nv && c + 1 < chunks) ga__eg_join_run(L, dtable, key, c, size, chunks, v, mine, step);
}
#endif
