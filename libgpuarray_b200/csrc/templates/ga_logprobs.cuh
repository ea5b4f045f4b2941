/* Log probabilities of given tokens, entropy and the most likely alternatives
 * of rows of logits, and the gradient of the first two.
 *
 * With x_j = scale * z_j, m = max z, S = sum_j e^(x_j - scale m):
 *   logp    = scale (z_t - m) - ln S
 *   entropy = ln S - (1/S) sum_j e^(x_j - scale m) (x_j - scale m)
 *   dz_j    = scale (a (1[j = t] - p_j) - b p_j (ln p_j + entropy)),
 *             p_j = e^(x_j - scale m - ln S), a and b the gradients arriving
 *             at logp and entropy.
 * One pass over a row keeps (m, S, T = sum e y) with y in powers of two and
 * rescales S and T when m grows (Milakov and Gimelshein, online softmax).
 * Differences to m are taken before the scale is applied, so that logits of
 * the type's lowest value, and rows of nothing else, stay finite.
 *   a row without a logit above -inf: logp and alternatives -inf, entropy 0,
 *     gradient 0;   a row with a NaN or +inf: NaN everywhere.
 *
 * Defines needed: GA_LP_BUILD_ROWS or GA_LP_BUILD_GRAD, GA_LP_Z_T (logits),
 * GA_LP_ZTYPE (0 half, 1 float), GA_LP_G_T and GA_LP_GTYPE (dlogits),
 * GA_LP_I_T (token ids), GA_LP_ND (leading dimensions), GA_LP_CONTIG (elements
 * of a row adjacent), GA_LP_ENT (entropy wanted), and for the rows kernel
 * GA_LP_FOLD (see ga__lp_step), GA_LP_THREADS, GA_LP_GROUP (threads per row: 32 or GA_LP_THREADS),
 * GA_LP_CLUSTER (CTAs per row), GA_LP_TOP (alternatives wanted). */
#include "ga_lm_common.cuh"

#define GA_LP_LOG2E 1.4426950408889634f
#define GA_LP_LN2 0.6931471805599453f

struct ga__lp_layout {
  unsigned long long rows;
  unsigned int v;   /* logits in a row, < 2^31 */
  unsigned int top; /* alternatives */
  float scale;
  int has_ignore;
  long long ignore;
  unsigned long long dims[GA_LM_MAXD];
  long long z_str[GA_LM_MAXD], t_str[GA_LM_MAXD];
  long long z_col;
  /* rows kernel: logp, entropy, stats, top values, top ids; gradient: stats, dlogp, entropy,
   * dentropy, dlogits */
  long long o_str[5][GA_LM_MAXD];
  long long o_col[5];
};

#if GA_LP_CONTIG
#define GA_LP_E (16 / (int)sizeof(GA_LP_Z_T))
#else
#define GA_LP_E 1
#endif

/* A row as vectors of GA_LP_E elements at 16-byte boundaries: vector w holds elements
 * w * E - skip ... of the row, of which those below 0 and beyond v are not there. */
struct ga__lp_row {
  const char *z;
  const char *base;
  unsigned int skip, nv;
};

static __device__ __forceinline__ ga__lp_row ga__lp_open(const ga__lp_layout &L, const char *logits,
                                                         unsigned long long row) {
  ga__lp_row r;
  r.z = logits + ga__lm_offset<GA_LP_ND>(row, L.dims, L.z_str);
#if GA_LP_CONTIG
  const unsigned int off = (unsigned int)((size_t)r.z & 15);
  r.base = r.z - off;
  r.skip = off / (unsigned int)sizeof(GA_LP_Z_T);
#else
  r.base = r.z;
  r.skip = 0;
#endif
  r.nv = (L.v + r.skip + GA_LP_E - 1) / GA_LP_E;
  return r;
}

/* one vector as 32-bit words (two halves or one float each) */
#if GA_LP_ZTYPE == 0
#define GA_LP_W ((GA_LP_E + 1) / 2)
#else
#define GA_LP_W GA_LP_E
#endif
struct alignas(GA_LP_CONTIG ? 16 : 4) ga__lp_words {
  unsigned int w[GA_LP_W];
};
#if GA_LP_ZTYPE == 0
#define GA_LP_MINUS_INF 0xfc00u
#else
#define GA_LP_MINUS_INF 0xff800000u
#endif

/* The elements that are not there read as -inf, which changes neither m nor S nor T. */
static __device__ __forceinline__ ga__lp_words ga__lp_load_part(const ga__lp_layout &L,
                                                                const ga__lp_row &r, unsigned int w) {
  ga__lp_words q;
#pragma unroll
  for (int j = 0; j < GA_LP_W; j++)
    q.w[j] = GA_LP_ZTYPE == 0 ? (GA_LP_MINUS_INF | GA_LP_MINUS_INF << 16) : GA_LP_MINUS_INF;
#pragma unroll
  for (int j = 0; j < GA_LP_E; j++) {
    const unsigned int i = w * GA_LP_E + j - r.skip; /* wraps below the row's start */
    if (i < L.v) {
#if GA_LP_ZTYPE == 0
      const unsigned int h = *reinterpret_cast<const unsigned short *>(r.z + (long long)i * L.z_col);
      q.w[j / 2] = (j & 1) ? (q.w[j / 2] & 0xffffu) | (h << 16) : (q.w[j / 2] & 0xffff0000u) | h;
#else
      q.w[j] = *reinterpret_cast<const unsigned int *>(r.z + (long long)i * L.z_col);
#endif
    }
  }
  return q;
}

static __device__ __forceinline__ int ga__lp_whole(const ga__lp_layout &L, const ga__lp_row &r,
                                                   unsigned int w) {
  return GA_LP_CONTIG && w * GA_LP_E >= r.skip && (w + 1) * GA_LP_E - r.skip <= L.v;
}

static __device__ __forceinline__ ga__lp_words ga__lp_load(const ga__lp_layout &L, const ga__lp_row &r,
                                                           unsigned int w) {
  if (ga__lp_whole(L, r, w))
    return *reinterpret_cast<const ga__lp_words *>(r.base + (size_t)w * 16);
  return ga__lp_load_part(L, r, w);
}

/* A CTA's vectors [v0, v1) of a row: those in [f0, f1) are whole, or elements apart by themselves;
 * the row's first or last one may be a part of a vector (GA_LP_NONE: it is not). The thread
 * `lane` of `group` has f0 + lane, f0 + lane + group ...; thread 0 also p0, thread 1 also p1. */
#define GA_LP_NONE 0xffffffffu
struct ga__lp_share {
  unsigned int v0, v1, f0, f1, p0, p1;
};
static __device__ __forceinline__ ga__lp_share ga__lp_split(const ga__lp_layout &L, const ga__lp_row &r,
                                                            unsigned int part, unsigned int parts) {
  ga__lp_share s;
  const unsigned int each = (r.nv + parts - 1) / parts;
  s.v0 = part * each < r.nv ? part * each : r.nv;
  s.v1 = r.nv - s.v0 < each ? r.nv : s.v0 + each;
  s.f0 = s.v0;
  s.f1 = s.v1;
  s.p0 = s.p1 = GA_LP_NONE;
  if (s.v0 < s.v1 && s.v0 == 0 && r.skip > 0) s.p0 = s.f0++;
  if (s.f0 < s.f1 && s.v1 == r.nv && r.nv * GA_LP_E - r.skip > L.v) s.p1 = --s.f1;
  return s;
}
static __device__ __forceinline__ unsigned int ga__lp_extra(const ga__lp_share &s, unsigned int lane) {
  return lane == 0 ? s.p0 : lane == 1 ? s.p1 : GA_LP_NONE;
}
/* one of [f0, f1) */
static __device__ __forceinline__ ga__lp_words ga__lp_load_whole(const ga__lp_layout &L, const ga__lp_row &r,
                                                                 unsigned int w) {
  if (GA_LP_CONTIG) return *reinterpret_cast<const ga__lp_words *>(r.base + (size_t)w * 16);
  return ga__lp_load_part(L, r, w);
}

static __device__ __forceinline__ float ga__lp_z(const char *p) {
#if GA_LP_ZTYPE == 0
  return ga_half2float(*reinterpret_cast<const ga_half *>(p));
#else
  return *reinterpret_cast<const float *>(p);
#endif
}

/* pair k of the vector as two floats (the second -inf where a vector has one element) */
#define GA_LP_PAIRS ((GA_LP_E + 1) / 2)
static __device__ __forceinline__ void ga__lp_pair(const ga__lp_words &q, int k, float &a, float &b) {
#if GA_LP_ZTYPE == 0
  ga__unpack_h2(q.w[k], a, b);
#else
  a = __uint_as_float(q.w[2 * k]);
  b = 2 * k + 1 < GA_LP_W ? __uint_as_float(q.w[2 * k + 1 < GA_LP_W ? 2 * k + 1 : 0])
                          : __uint_as_float(0xff800000u);
#endif
}

#ifdef GA_LP_BUILD_ROWS
#define GA_LP_U 4 /* vectors of a thread in one step, and as many fetched ahead */
#define GA_LP_CAND (GA_LP_GROUP == 32 ? 256 : 512)
/* below every logit that is not -inf: the maximum of nothing (a half is never so low; a float
 * logit of exactly this value gives the right S all the same) */
#define GA_LP_NOTHING -3.402823466e38f
/* 2^y is 0 from here on; keeps 0 * y finite */
#define GA_LP_YMIN -200.0f

struct ga__lp_state {
  float m, s, t;
};

/* The states of `width` lanes (a power of two) as one, the same bits in each of them. */
static __device__ __forceinline__ ga__lp_state ga__lp_merge(ga__lp_state a, float c, int width) {
  float m = a.m;
#pragma unroll
  for (int d = width / 2; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  const float d = ga__max_nan((a.m - m) * c, GA_LP_YMIN), f = ga__ex2(d);
  a.t = (a.t + a.s * d) * f;
  a.s *= f;
  a.m = m;
#pragma unroll
  for (int d = width / 2; d > 0; d /= 2) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, d);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, d);
  }
  return a;
}

/* the largest element of N vectors, NaNs left out where there are numbers */
template <int N>
static __device__ __forceinline__ float ga__lp_max(const ga__lp_words q[N]) {
#if GA_LP_ZTYPE == 0
  unsigned int h = q[0].w[0];
#pragma unroll
  for (int j = 1; j < N * GA_LP_W; j++) h = ga__max_h2(h, q[j / GA_LP_W].w[j % GA_LP_W]);
  float a, b;
  ga__unpack_h2(h, a, b);
  return fmaxf(a, b);
#else
  float a = __uint_as_float(q[0].w[0]);
#pragma unroll
  for (int j = 1; j < N * GA_LP_W; j++) a = fmaxf(a, __uint_as_float(q[j / GA_LP_W].w[j % GA_LP_W]));
  return a;
#endif
}

/* N vectors into a thread's state: the sums are kept in pairs beside it. Returns their largest.
 *
 * GA_LP_FOLD (halfs, a scale of at most 64): y = z c - mc by one fused operation, mc = m c
 * rounded (by itself, not inside another fused operation). All terms are then off by the same factor 2^d, d = m c - mc exactly, |d| < 1/2, which
 * ga__lp_settle takes back once. Otherwise y = (z - m) c. */
template <int N>
static __device__ __forceinline__ float ga__lp_step(const ga__lp_words q[N], float c, ga__lp_state &st,
                                                    ga__f2 &s2, ga__f2 &t2) {
  const float top = ga__lp_max<N>(q);
  if (top > st.m) {
#if GA_LP_FOLD
    const float d = st.m == GA_LP_NOTHING ? GA_LP_YMIN : ga__max_nan(__fmul_rn(st.m, c) - __fmul_rn(top, c), GA_LP_YMIN);
#else
    const float d = ga__max_nan((st.m - top) * c, GA_LP_YMIN);
#endif
    const float f = ga__ex2(d);
    const ga__f2 f2 = ga__f2_of(f, f);
#if GA_LP_ENT
    t2 = ga__f2_mul(ga__f2_fma(s2, ga__f2_of(d, d), t2), f2);
#endif
    s2 = ga__f2_mul(s2, f2);
    st.m = top;
  }
  const ga__f2 c2 = ga__f2_of(c, c);
#if GA_LP_FOLD
  const float mc = st.m == GA_LP_NOTHING ? 0.0f : -__fmul_rn(st.m, c);
  const ga__f2 mc2 = ga__f2_of(mc, mc);
#else
  const ga__f2 m2 = ga__f2_of(-st.m, -st.m);
#endif
#pragma unroll
  for (int u = 0; u < N; u++)
#pragma unroll
    for (int k = 0; k < GA_LP_PAIRS; k++) {
      float a, b;
      ga__lp_pair(q[u], k, a, b);
#if GA_LP_FOLD
      ga__f2_to(ga__f2_fma(ga__f2_of(a, b), c2, mc2), a, b);
#else
      ga__f2_to(ga__f2_mul(ga__f2_add(ga__f2_of(a, b), m2), c2), a, b);
#endif
#if GA_LP_ENT
      a = ga__max_nan(a, GA_LP_YMIN); /* e y is 0 for a logit of -inf */
      b = ga__max_nan(b, GA_LP_YMIN);
#endif
      const ga__f2 e2 = ga__f2_of(ga__ex2(a), ga__ex2(b));
      s2 = ga__f2_add(s2, e2);
#if GA_LP_ENT
      t2 = ga__f2_fma(e2, ga__f2_of(a, b), t2);
#endif
    }
  return top;
}

/* The thread's sums, relative to its m. */
static __device__ __forceinline__ void ga__lp_settle(float c, ga__lp_state &st, ga__f2 s2, ga__f2 t2) {
  float a, b;
  ga__f2_to(s2, a, b);
  st.s = a + b;
  ga__f2_to(t2, a, b);
  st.t = a + b;
#if GA_LP_FOLD
  if (st.m != GA_LP_NOTHING) {
    const float mc = __fmul_rn(st.m, c), d = fmaf(st.m, c, -mc), f = ga__ex2(-d);
    st.t = (st.t - st.s * d) * f;
    st.s *= f;
  }
#endif
}

#if GA_LP_TOP
/* Orders by value, NaN lowest, and among equal values the lower index higher; 0 is no element. */
static __device__ __forceinline__ unsigned long long ga__lp_key(float z, unsigned int i) {
  unsigned int b = __float_as_uint(z + 0.0f); /* -0 and +0 are one value */
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (z != z) b = 0;
  return ((unsigned long long)b << 32) | (0xffffffffu - i);
}
static __device__ __forceinline__ float ga__lp_key_value(unsigned long long k) {
  const unsigned int b = (unsigned int)(k >> 32);
  if (b == 0) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

/* keys of the vector's elements that are there; absent ones 0 */
static __device__ __forceinline__ void ga__lp_keys(const ga__lp_layout &L, const ga__lp_row &r,
                                                   unsigned int w, unsigned long long k[2 * GA_LP_PAIRS]) {
  const ga__lp_words q = ga__lp_load(L, r, w);
#pragma unroll
  for (int p = 0; p < GA_LP_PAIRS; p++) {
    float z[2];
    ga__lp_pair(q, p, z[0], z[1]);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const unsigned int i = w * GA_LP_E + 2 * p + h - r.skip;
      k[2 * p + h] = (2 * p + h < GA_LP_E && i < L.v) ? ga__lp_key(z[h], i) : 0;
    }
  }
}

/* The vector's largest key where it holds a value of m or more, else 0. */
static __device__ __forceinline__ unsigned long long ga__lp_best(const ga__lp_layout &L, const ga__lp_row &r,
                                                                 unsigned int w, float m) {
  unsigned long long k[2 * GA_LP_PAIRS], best = 0;
  const ga__lp_words q = ga__lp_load(L, r, w);
  if (!(ga__lp_max<1>(&q) >= m)) return 0;
  ga__lp_keys(L, r, w, k);
#pragma unroll
  for (int j = 0; j < 2 * GA_LP_PAIRS; j++) best = k[j] > best ? k[j] : best;
  return best;
}

/* the threads of a row meet */
static __device__ __forceinline__ void ga__lp_sync() {
  if (GA_LP_GROUP == 32) __syncwarp();
  else __syncthreads();
}

/* A thread's vectors in pieces of so many steps of GA_LP_U, that GA_LP_PIECES hold them all; what
 * is left over after its whole steps and the extra vector belong to the piece of the next step. */
#define GA_LP_PIECES (GA_LP_GROUP == 32 ? 16 : 2048 / GA_LP_GROUP)
static __device__ __forceinline__ unsigned int ga__lp_piece_steps(const ga__lp_share &s) {
  const unsigned int steps = (s.f1 - s.f0) / (GA_LP_U * GA_LP_GROUP) + 2; /* of any thread, at most */
  return (steps + GA_LP_PIECES - 1) / GA_LP_PIECES;
}
/* the last piece of thread t */
static __device__ __forceinline__ unsigned int ga__lp_last_piece(const ga__lp_share &s, unsigned int t) {
  const unsigned int mine = s.f0 + t < s.f1 ? (s.f1 - s.f0 - t + GA_LP_GROUP - 1) / GA_LP_GROUP : 0;
  return mine / GA_LP_U / ga__lp_piece_steps(s);
}

struct ga__lp_top_smem {
  unsigned long long cand[GA_LP_CAND];
  unsigned long long best[GA_LP_GROUP];
  unsigned long long out[GA_LP_CLUSTER * 32]; /* the CTAs' lists, in the first CTA of a cluster */
  unsigned long long tau;
  unsigned int high[GA_LP_GROUP];
  unsigned int piece[GA_LP_PIECES][GA_LP_GROUP]; /* largest values of the threads' pieces */
  unsigned int list[GA_LP_CAND];                   /* piece * GA_LP_GROUP + thread */
  unsigned int vec[GA_LP_CAND];
  unsigned int nlist, nvec, ncand, count;
};

/* The top-th largest of the lanes' keys, at least 1 (0: no key); the same in every lane. */
template <typename K>
static __device__ __forceinline__ K ga__lp_nth(K mine, unsigned int top) {
  const unsigned int lane = threadIdx.x % 32;
  unsigned int place = 0;
#pragma unroll
  for (int j = 0; j < 32; j++) {
    const K o = __shfl_sync(0xffffffffu, mine, j);
    place += o > mine || (o == mine && j < (int)lane);
  }
  const unsigned int who = __ballot_sync(0xffffffffu, place == top - 1);
  const K t = __shfl_sync(0xffffffffu, mine, __ffs(who) - 1);
  return t > 0 ? t : 1;
}

static __device__ __forceinline__ void ga__lp_list(unsigned int piece, ga__lp_top_smem &S) {
  const unsigned int at = atomicAdd(&S.nlist, 1u);
  if (at < GA_LP_CAND) S.list[at] = piece * GA_LP_GROUP + threadIdx.x % GA_LP_GROUP;
}
static __device__ __forceinline__ void ga__lp_append(unsigned long long key, ga__lp_top_smem &S) {
  const unsigned int at = atomicAdd(&S.ncand, 1u);
  if (at < GA_LP_CAND) S.cand[at] = key;
}

/* Appends the keys from `tau` on of the listed pieces' vectors to the candidates: first the vectors
 * that hold one, by their largest element, then an element for each thread. */
static __device__ __forceinline__ void ga__lp_collect(const ga__lp_layout &L, const ga__lp_row &r,
                                                      const ga__lp_share &sh, unsigned long long tau,
                                                      ga__lp_top_smem &S) {
  const unsigned int steps = ga__lp_piece_steps(sh);
  const unsigned int per = steps * GA_LP_U + 1; /* and the extra vector */
  const unsigned int items = (S.nlist < GA_LP_CAND ? S.nlist : GA_LP_CAND) * per;
  const float inv = 1.0f / (float)per; /* exact quotients below 2^20 */
  const unsigned int tid = threadIdx.x % GA_LP_GROUP;
  if (tid == 0 && S.nlist > GA_LP_CAND) S.nvec = GA_LP_CAND + 1;
  for (unsigned int it = tid; it < items && S.nlist <= GA_LP_CAND; it += GA_LP_GROUP) {
    if (*(volatile unsigned int *)&S.nvec > GA_LP_CAND) break; /* too many: they are not used */
    const unsigned int l = items < (1u << 20) ? (unsigned int)(((float)it + 0.5f) * inv) : it / per;
    const unsigned int t = S.list[l] % GA_LP_GROUP, p = S.list[l] / GA_LP_GROUP, j = it - l * per;
    unsigned int w;
    if (j + 1 < per) {
      w = sh.f0 + t + (p * steps * GA_LP_U + j) * GA_LP_GROUP;
      if (w >= sh.f1) continue;
    } else { /* the extra vector is in the last piece of its thread that there is */
      w = ga__lp_extra(sh, t);
      if (w == GA_LP_NONE || p != ga__lp_last_piece(sh, t)) continue;
    }
    const ga__lp_words q = ga__lp_load(L, r, w);
    /* no element's key is above that of the largest value at the vector's first place */
    const unsigned int i0 = w * GA_LP_E < r.skip ? 0 : w * GA_LP_E - r.skip;
    if (ga__lp_key(ga__lp_max<1>(&q), i0) >= tau) {
      const unsigned int at = atomicAdd(&S.nvec, 1u);
      if (at < GA_LP_CAND) S.vec[at] = w;
    }
  }
  ga__lp_sync();
  if (S.nvec > GA_LP_CAND) { /* the same in every thread */
    if (tid == 0) S.ncand = GA_LP_CAND + 1;
  } else {
    const unsigned int elements = S.nvec * GA_LP_E;
    for (unsigned int it = tid; it < elements; it += GA_LP_GROUP) {
      const unsigned int i = S.vec[it / GA_LP_E] * GA_LP_E + it % GA_LP_E - r.skip;
      if (i >= L.v) continue;
      const unsigned long long k = ga__lp_key(ga__lp_z(r.z + (long long)i * L.z_col), i);
      if (k >= tau) ga__lp_append(k, S);
    }
  }
  ga__lp_sync();
}

/* The `top` largest keys of a CTA's vectors of the row, into out[0..32) of this CTA's or the
 * cluster's first CTA's shared memory (0 where there are fewer). All threads of the group, after a
 * barrier behind which S.high has every thread's largest value and the counters are 0; m: this
 * thread's.
 *
 * The largest values of 32 disjoint groups of threads are values of 32 elements, so the top-th
 * largest of them, tau, is a lower bound for the top-th largest of all, and every element that
 * reaches it belongs to a piece of a thread whose largest does: only those pieces are read again.
 * (For 20 alternatives of 256 threads they are about 30.) Where more elements reach tau than can
 * be held (equal values: rows with fewer numbers than alternatives, constants), the same is done
 * with keys that break ties by the index; where that is still too much (a row that hides its
 * largest elements in few threads' vectors) or NaNs are about (`odd`), tau is found by halving
 * over the row. */
static __device__ void ga__lp_top(const ga__lp_layout &L, const ga__lp_row &r, const ga__lp_share &sh,
                                  float m, int odd, ga__lp_top_smem &S) {
  const unsigned int tid = threadIdx.x % GA_LP_GROUP, lane = tid % 32;
  const unsigned int last = ga__lp_last_piece(sh, tid);
  unsigned long long k[2 * GA_LP_PAIRS], tau = 0;
  if (!odd) {
    if (tid < 32) {
      unsigned int high = 0;
#pragma unroll
      for (int j = 0; j < GA_LP_GROUP / 32; j++) {
        const unsigned int b = S.high[j * 32 + lane];
        high = b > high ? b : high;
      }
      high = ga__lp_nth(high, L.top);
      if (lane == 0) S.tau = (unsigned long long)high << 32;
    }
    ga__lp_sync();
    tau = S.tau;
    const float minus_inf = __uint_as_float(0xff800000u);
    const int few = (tau >> 32) == (ga__lp_key(minus_inf, 0) >> 32); /* fewer above -inf than asked for */
    if (!few) {
      if (S.high[tid] > 0 && ga__lp_key(m, 0) >= tau)
        for (unsigned int p = 0; p <= last; p++)
          if ((unsigned long long)S.piece[p][tid] << 32 >= tau) ga__lp_list(p, S);
      ga__lp_sync();
      ga__lp_collect(L, r, sh, tau, S);
    }
    if (few || S.ncand > GA_LP_CAND) { /* the same in every thread */
      unsigned long long mine = 0;
      /* its first place: p0 is before the whole vectors, p1 behind them */
      if (tid == 0 && sh.p0 != GA_LP_NONE) mine = ga__lp_best(L, r, sh.p0, m);
      for (unsigned int w = sh.f0 + tid; mine == 0 && w < sh.f1; w += GA_LP_GROUP) mine = ga__lp_best(L, r, w, m);
      if (mine == 0 && tid == 1 && sh.p1 != GA_LP_NONE) mine = ga__lp_best(L, r, sh.p1, m);
      S.best[tid] = mine;
      ga__lp_sync();
      if (tid == 0) S.nlist = S.nvec = S.ncand = 0;
      unsigned long long most = 0;
#pragma unroll
      for (int j = 0; j < GA_LP_GROUP / 32; j++) {
        const unsigned long long b = S.best[j * 32 + lane];
        most = b > most ? b : most;
      }
      tau = ga__lp_nth(most, L.top);
      ga__lp_sync();
      if (mine >= tau)
        for (unsigned int p = 0; p <= last; p++) ga__lp_list(p, S);
      ga__lp_sync();
      ga__lp_collect(L, r, sh, tau, S);
    }
  }
  if (odd || S.ncand > GA_LP_CAND) { /* the same in every thread */
    /* the first count is of all there is; after it fewer than `top` keys reach hi and at least as
     * many lo, and keys differ: 64 halvings end with exactly `top` */
    unsigned long long lo = 1, hi = ~0ULL; /* above every key: the largest value, inf, has 0xff800000 */
    for (int step = 0; step < 66; step++) {
      const unsigned long long mid = step == 0 ? 1 : lo + (hi - lo) / 2;
      unsigned int c = 0;
      ga__lp_sync();
      if (tid == 0) S.count = 0;
      ga__lp_sync();
      for (unsigned int w = sh.v0 + tid; w < sh.v1; w += GA_LP_GROUP) {
        ga__lp_keys(L, r, w, k);
#pragma unroll
        for (int j = 0; j < 2 * GA_LP_PAIRS; j++) c += k[j] >= mid;
      }
      c = ga__warp_sum_u32(c);
      if (lane == 0) atomicAdd(&S.count, c);
      ga__lp_sync();
      c = S.count;
      if (c >= L.top || step == 0) lo = mid;
      else hi = mid;
      if (c <= GA_LP_CAND && (c >= L.top || step == 0)) break;
    }
    tau = lo;
    if (tid == 0) S.ncand = 0;
    ga__lp_sync();
    for (unsigned int w = sh.v0 + tid; w < sh.v1; w += GA_LP_GROUP) {
      ga__lp_keys(L, r, w, k);
#pragma unroll
      for (int j = 0; j < 2 * GA_LP_PAIRS; j++)
        if (k[j] >= tau) ga__lp_append(k[j], S);
    }
    ga__lp_sync();
  }
  /* a key's place is the number of larger ones */
  const unsigned int n = S.ncand < GA_LP_CAND ? S.ncand : GA_LP_CAND;
#if GA_LP_CLUSTER > 1
  const unsigned int slot = ga__cluster_rank() * 32;
  for (unsigned int i = tid + n; i < L.top; i += GA_LP_GROUP) ga__cluster_put(&S.out[slot + i], 0, 0ULL);
#else
  for (unsigned int i = tid + n; i < L.top; i += GA_LP_GROUP) S.out[i] = 0;
#endif
  for (unsigned int i = tid; i < n; i += GA_LP_GROUP) {
    const unsigned long long key = S.cand[i];
    unsigned int place = 0;
#pragma unroll 4
    for (unsigned int j = 0; j < n; j++) place += S.cand[j] > key;
    if (place < L.top) {
#if GA_LP_CLUSTER > 1
      ga__cluster_put(&S.out[slot + place], 0, key);
#else
      S.out[place] = key;
#endif
    }
  }
}
#endif

struct ga__lp_shared {
#if GA_LP_TOP
  ga__lp_top_smem tops[GA_LP_THREADS / GA_LP_GROUP];
#endif
  unsigned long long parts[GA_LP_CLUSTER][2]; /* the CTAs' states, in the first CTA of a cluster */
  ga__lp_state warps[GA_LP_THREADS / 32];
};

extern "C" __global__ void __launch_bounds__(GA_LP_THREADS, 1024 / GA_LP_THREADS)
#if GA_LP_CLUSTER > 1
    __cluster_dims__(GA_LP_CLUSTER, 1, 1)
#endif
ga_lp_rows(const __grid_constant__ ga__lp_layout L, const char *logits, const char *targets,
           char *logp, char *entropy, char *stats, char *topv, char *topi, int *err) {
  ga__grid_dependency_sync();
  const unsigned int lane = threadIdx.x % GA_LP_GROUP;
#if GA_LP_CLUSTER > 1
  const unsigned long long row = blockIdx.x / GA_LP_CLUSTER;
  const unsigned int part = ga__cluster_rank();
#else
  const unsigned long long row =
      (unsigned long long)blockIdx.x * (GA_LP_THREADS / GA_LP_GROUP) + threadIdx.x / GA_LP_GROUP;
  const unsigned int part = 0;
#if GA_LP_GROUP < GA_LP_THREADS
  if (row >= L.rows) return; /* a whole warp; nothing below waits for another */
#endif
#endif
#if GA_LP_CLUSTER > 1
  ga__cluster_arrive(); /* waited for before the first store to another CTA's shared memory */
#endif
  const ga__lp_row r = ga__lp_open(L, logits, row);
  const ga__lp_share my = ga__lp_split(L, r, part, GA_LP_CLUSTER);
  const float c = L.scale * GA_LP_LOG2E;

  /* the target's logit is fetched while the row streams */
  long long target = -1;
  float zt = 0;
  if (lane == 0 && part == 0 && logp != nullptr) {
    target = (long long)*reinterpret_cast<const GA_LP_I_T *>(
        targets + ga__lm_offset<GA_LP_ND>(row, L.dims, L.t_str));
    if (target >= 0 && target < (long long)L.v) zt = ga__lp_z(r.z + target * L.z_col);
  }

  ga__lp_state st = {GA_LP_NOTHING, 0.0f, 0.0f};
  ga__f2 s2 = ga__f2_of(0.0f, 0.0f), t2 = s2;
  const unsigned int extra = ga__lp_extra(my, lane);
  unsigned int w = my.f0 + lane;
  GA_LM_SHARED(ga__lp_shared, sh);
#if GA_LP_TOP
  ga__lp_top_smem &tops = sh.tops[threadIdx.x / GA_LP_GROUP];
  const unsigned int steps = ga__lp_piece_steps(my);
  unsigned int left = steps, piece = 0;
  float largest = __uint_as_float(0xff800000u); /* of the piece */
#endif
  /* the next vectors are fetched before the present ones are worked on */
  ga__lp_words next[GA_LP_U];
  int more = w + (GA_LP_U - 1) * GA_LP_GROUP < my.f1;
  if (more) {
#pragma unroll
    for (int u = 0; u < GA_LP_U; u++) next[u] = ga__lp_load_whole(L, r, w + u * GA_LP_GROUP);
  }
  while (more) {
    ga__lp_words q[GA_LP_U];
#pragma unroll
    for (int u = 0; u < GA_LP_U; u++) q[u] = next[u];
    w += GA_LP_U * GA_LP_GROUP;
    more = w + (GA_LP_U - 1) * GA_LP_GROUP < my.f1;
    if (more) {
#pragma unroll
      for (int u = 0; u < GA_LP_U; u++) next[u] = ga__lp_load_whole(L, r, w + u * GA_LP_GROUP);
    }
    const float top = ga__lp_step<GA_LP_U>(q, c, st, s2, t2);
#if GA_LP_TOP
    largest = fmaxf(largest, top);
    if (--left == 0) {
      tops.piece[piece++][lane] = (unsigned int)(ga__lp_key(largest, 0) >> 32);
      largest = __uint_as_float(0xff800000u);
      left = steps;
    }
#endif
  }
  { /* fewer than GA_LP_U are left: all of them in flight, then one at a time */
    ga__lp_words q[GA_LP_U];
#pragma unroll
    for (int u = 0; u + 1 < GA_LP_U; u++)
      if (w + u * GA_LP_GROUP < my.f1) q[u] = ga__lp_load_whole(L, r, w + u * GA_LP_GROUP);
    if (extra != GA_LP_NONE) q[GA_LP_U - 1] = ga__lp_load_part(L, r, extra);
#pragma unroll 1
    for (int u = 0; u < GA_LP_U; u++) {
      if (u + 1 < GA_LP_U ? w + u * GA_LP_GROUP < my.f1 : extra != GA_LP_NONE) {
        const float top = ga__lp_step<1>(&q[0], c, st, s2, t2);
#if GA_LP_TOP
        largest = fmaxf(largest, top);
#endif
      }
#pragma unroll
      for (int i = 0; i + 1 < GA_LP_U; i++) q[i] = q[i + 1];
    }
  }
#if GA_LP_TOP
  tops.piece[piece][lane] = (unsigned int)(ga__lp_key(largest, 0) >> 32);
#endif
  ga__lp_settle(c, st, s2, t2);
#if GA_LP_TOP
  const float most = st.s == 0.0f ? __uint_as_float(0xff800000u) : st.m; /* this thread's largest */
  tops.high[lane] =
      my.f0 + lane < my.f1 || extra != GA_LP_NONE ? (unsigned int)(ga__lp_key(most, 0) >> 32) : 0;
  if (lane == 0) tops.nlist = tops.nvec = tops.ncand = 0;
#endif
  st = ga__lp_merge(st, c, 32);
#if GA_LP_GROUP > 32
  if (threadIdx.x % 32 == 0) sh.warps[threadIdx.x / 32] = st;
  __syncthreads();
  st = ga__lp_merge(sh.warps[threadIdx.x % (GA_LP_THREADS / 32)], c, GA_LP_THREADS / 32);
#elif GA_LP_TOP
  __syncwarp();
#endif
#if GA_LP_CLUSTER > 1
  ga__cluster_wait(); /* every CTA of the cluster runs */
#endif
#if GA_LP_TOP
  ga__lp_top(L, r, my, most, !(st.s == st.s), tops);
#endif
#if GA_LP_CLUSTER > 1
  /* the CTAs' states and lists meet in the first one */
  if (threadIdx.x == 0) {
    ga__cluster_put(&sh.parts[part][0], 0, (unsigned long long)__float_as_uint(st.m) << 32 | __float_as_uint(st.s));
    ga__cluster_put(&sh.parts[part][1], 0, (unsigned long long)__float_as_uint(st.t));
  }
  ga__cluster_arrive();
  ga__cluster_wait();
  if (part != 0) return;
  {
    const unsigned int i = threadIdx.x % GA_LP_CLUSTER;
    st.m = __uint_as_float((unsigned int)(sh.parts[i][0] >> 32));
    st.s = __uint_as_float((unsigned int)sh.parts[i][0]);
    st.t = __uint_as_float((unsigned int)sh.parts[i][1]);
    st = ga__lp_merge(st, c, GA_LP_CLUSTER);
  }
#endif
  const int empty = st.s == 0.0f;
  const float ls = logf(st.s);
  const float minus_inf = __uint_as_float(0xff800000u);
  if (lane == 0) {
    if (logp != nullptr) {
      float p;
      if (L.has_ignore && target == L.ignore) p = 0.0f;
      else if (target < 0 || target >= (long long)L.v) {
        p = __uint_as_float(0x7fffffffu);
        if (err != nullptr) *err = -1;
      } else p = empty ? minus_inf : (zt - st.m) * L.scale - ls;
      *reinterpret_cast<float *>(logp + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[0])) = p;
    }
#if GA_LP_ENT
    if (entropy != nullptr) {
      const float h = ls - GA_LP_LN2 * (st.t / st.s);
      *reinterpret_cast<float *>(entropy + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[1])) =
          empty || h < 0.0f ? 0.0f : h;
    }
#endif
    if (stats != nullptr) {
      char *p = stats + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[2]);
      /* m leaves NaNs out: the sum tells */
      *reinterpret_cast<float *>(p) = empty ? minus_inf : st.s == st.s ? st.m : st.s;
      *reinterpret_cast<float *>(p + L.o_col[2]) = ls;
    }
  }
#if GA_LP_TOP
#if GA_LP_CLUSTER > 1
  const unsigned int n = GA_LP_CLUSTER * 32;
#else
  ga__lp_sync();
  const unsigned int n = L.top;
#endif
  for (unsigned int i = lane; i < n; i += GA_LP_GROUP) {
#if GA_LP_CLUSTER > 1
    if (i % 32 >= L.top) continue;
#endif
    const unsigned long long key = tops.out[i];
    if (key == 0) continue;
    unsigned int place = i;
#if GA_LP_CLUSTER > 1
    place = 0;
    for (unsigned int l = 0; l < GA_LP_CLUSTER; l++)
#pragma unroll 4
      for (unsigned int j = 0; j < L.top; j++) place += tops.out[l * 32 + j] > key;
    if (place >= L.top) continue;
#endif
    if (topv != nullptr)
      *reinterpret_cast<float *>(topv + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[3]) +
                                 place * L.o_col[3]) =
          empty ? minus_inf : (ga__lp_key_value(key) - st.m) * L.scale - ls;
    if (topi != nullptr)
      *reinterpret_cast<GA_LP_I_T *>(topi + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[4]) +
                                     place * L.o_col[4]) =
          (GA_LP_I_T)(0xffffffffu - (unsigned int)key);
  }
#endif
}
#endif

#ifdef GA_LP_BUILD_GRAD
#define GA_LP_U 4

/* Elements i ... of the gradient's row: all of a vector's, or those from `skip` on that the row of
 * n has. */
static __device__ __forceinline__ void ga__lp_store(char *g, long long col, long long i, unsigned int skip,
                                                    unsigned int n, const float x[2 * GA_LP_PAIRS],
                                                    int whole) {
  typedef ga__lm_vec<GA_LP_G_T, GA_LP_E> vec;
  char *p = g + i * col;
  if (whole && col == (long long)sizeof(GA_LP_G_T) && ((size_t)p & (alignof(vec) - 1)) == 0) {
    vec q;
    ga__lm_put<GA_LP_G_T, GA_LP_E>(q, x);
    ga__lm_store(p, q);
    return;
  }
#pragma unroll
  for (int j = 0; j < GA_LP_E; j++)
    if (j >= (int)skip && i + j < (long long)n) {
      ga__lm_vec<GA_LP_G_T, 1> q;
      ga__lm_put<GA_LP_G_T, 1>(q, x + j);
      ga__lm_store(p + j * col, q);
    }
}

/* A CTA walks a part of a row (blockDim.y rows where they are short), GA_LP_U vectors of a thread
 * at a time, the next ones fetched before the present ones are written. The row's numbers come from
 * the forward pass, so that the logits are read once and the gradient written once: bound by
 * memory. The last rows come first: they are what the forward pass left in L2. dlogits may be the
 * logits. */
static __device__ __forceinline__ void ga__lp_fetch(const ga__lp_layout &L, const ga__lp_row &r,
                                                    unsigned int w0, ga__lp_words q[GA_LP_U]) {
  const unsigned int end = w0 + (GA_LP_U - 1) * blockDim.x;
  if (GA_LP_CONTIG && w0 > 0 && end + 1 < r.nv) { /* neither the row's first nor its last vector */
#pragma unroll
    for (int u = 0; u < GA_LP_U; u++)
      q[u] = *reinterpret_cast<const ga__lp_words *>(r.base + (size_t)(w0 + u * blockDim.x) * 16);
    return;
  }
#pragma unroll
  for (int u = 0; u < GA_LP_U; u++)
    if (w0 + u * blockDim.x < r.nv) q[u] = ga__lp_load(L, r, w0 + u * blockDim.x);
}

extern "C" __global__ void __launch_bounds__(256)
ga_lp_grad(const __grid_constant__ ga__lp_layout L, char *dlogits, const char *logits,
           const char *targets, const char *stats, const char *dlogp, const char *entropy,
           const char *dentropy, int *err) {
  ga__grid_dependency_sync();
  const unsigned long long back = (unsigned long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (back >= L.rows) return;
  const unsigned long long row = L.rows - 1 - back;
  const ga__lp_row r = ga__lp_open(L, logits, row);
  unsigned int w0 = blockIdx.y * blockDim.x * GA_LP_U + threadIdx.x;
  if (w0 >= r.nv) return;
  char *g = dlogits + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[4]);

  long long target = (long long)*reinterpret_cast<const GA_LP_I_T *>(
      targets + ga__lm_offset<GA_LP_ND>(row, L.dims, L.t_str));
  const char *sp = stats + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[0]);
  const float m = *reinterpret_cast<const float *>(sp);
  const float ls = *reinterpret_cast<const float *>(sp + L.o_col[0]);
  float a = *reinterpret_cast<const float *>(dlogp + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[1]));
  int none = 0; /* the row's gradient is `fill` throughout */
  float fill = 0.0f;
  if (L.has_ignore && target == L.ignore) {
    a = 0.0f;
    target = -1;
    none = !GA_LP_ENT;
  } else if (target < 0 || target >= (long long)L.v) {
    a = fill = __uint_as_float(0x7fffffffu);
    if (w0 == 0 && err != nullptr) *err = -1;
  }
  if (m == __uint_as_float(0xff800000u)) none = 1; /* nothing above -inf in the row */
  const float c = L.scale * GA_LP_LOG2E;
  /* dz = e^(...) (w0 + w1 y) with y = log2 p, plus scale a at the target */
  float k0 = -L.scale * a, k1 = 0.0f;
#if GA_LP_ENT
  {
    const float b = *reinterpret_cast<const float *>(dentropy + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[3]));
    const float h = *reinterpret_cast<const float *>(entropy + ga__lm_offset<GA_LP_ND>(row, L.dims, L.o_str[2]));
    k0 -= L.scale * b * h;
    k1 = -L.scale * b * GA_LP_LN2;
  }
#endif
  const ga__f2 nm2 = ga__f2_of(-m, -m), c2 = ga__f2_of(c, c);
  const float l2 = -ls * GA_LP_LOG2E;
  const ga__f2 nl2 = ga__f2_of(l2, l2), k02 = ga__f2_of(k0, k0), k12 = ga__f2_of(k1, k1);
  const unsigned int step = gridDim.y * blockDim.x * GA_LP_U;
  ga__lp_words next[GA_LP_U];
  if (!none) ga__lp_fetch(L, r, w0, next);
  for (; w0 < r.nv; w0 += step) {
    ga__lp_words q[GA_LP_U];
#pragma unroll
    for (int u = 0; u < GA_LP_U; u++) q[u] = next[u];
    if (!none && w0 + step < r.nv) ga__lp_fetch(L, r, w0 + step, next);
#pragma unroll
    for (int u = 0; u < GA_LP_U; u++) {
      const unsigned int w = w0 + u * blockDim.x;
      if (w >= r.nv) break;
      float x[2 * GA_LP_PAIRS];
      if (none) {
#pragma unroll
        for (int j = 0; j < 2 * GA_LP_PAIRS; j++) x[j] = fill;
      } else {
#pragma unroll
        for (int k = 0; k < GA_LP_PAIRS; k++) {
          float p, s;
          ga__lp_pair(q[u], k, p, s);
          ga__f2_to(ga__f2_fma(ga__f2_add(ga__f2_of(p, s), nm2), c2, nl2), p, s);
          p = ga__max_nan(p, -200.0f);
          s = ga__max_nan(s, -200.0f);
          const ga__f2 y = ga__f2_of(p, s);
          const ga__f2 e = ga__f2_of(ga__ex2(p), ga__ex2(s));
          ga__f2_to(ga__f2_mul(e, ga__f2_fma(k12, y, k02)), x[2 * k], x[2 * k + 1]);
        }
        const unsigned int at = (unsigned int)target + r.skip - w * GA_LP_E;
        if (target >= 0 && at < GA_LP_E) {
#pragma unroll
          for (int j = 0; j < GA_LP_E; j++)
            if (at == j) x[j] += L.scale * a;
        }
      }
      const long long i = (long long)w * GA_LP_E - r.skip; /* below 0 where the row starts inside the vector */
      ga__lp_store(g, L.o_col[4], i, i < 0 ? r.skip : 0, L.v, x, ga__lp_whole(L, r, w));
    }
  }
}
#endif
