/* Token embedding and its gradient (include/gpuarray/embedding.h; kernels in
 * templates/ga_embed.cuh). */
#include <math.h>
#include "private.h"

typedef struct em_layout { /* the templates' ga__em_layout */
  unsigned long long n, v;
  unsigned int nv, chunk, chunks;
  int has_pad;
  long long pad;
  double scale;
  unsigned long long dims[GA_LM_MAXD];
  long long i_str[GA_LM_MAXD], t_str[GA_LM_MAXD];
  long long t_col, v_row, v_col;
} em_layout;

typedef struct eg_sort { /* the templates' ga__eg_sort */
  unsigned int n, tiles, tile, passes, pass;
} eg_sort;

struct _GpuEmbedGrad {
  gpucontext *ctx;
  ga_workspace ws;
};

static int is_real(int tc) { return tc == GA_HALF || tc == GA_FLOAT || tc == GA_DOUBLE; }

/* key: A type | O type << 8 | id type << 16 | E << 24 | ND << 32 | gradient << 40 |
 * accumulate << 41 | C << 48 | rounds of the one-launch sort << 56 | its CTAs << 60 */
static void emit(ga_strb *sb, uint64_t key) {
  const int a = (int)(key & 0xff), o = (int)((key >> 8) & 0xff), i = (int)((key >> 16) & 0xff);
  ga_strb_printf(sb,
                 "#include \"cluda.h\"\n#define %s\n#define GA_EM_A_T %s\n#define GA_EM_O_T %s\n"
                 "#define GA_EM_I_T %s\n#define GA_EM_F_T %s\n#define GA_EM_E %u\n"
                 "#define GA_EM_ND %u\n#define GA_EM_ACCUMULATE %u\n#define GA_EM_C %u\n"
                 "#define GA_EG_ROUNDS %u\n#define GA_EG_CLUSTER %u\n#include \"ga_embed.cuh\"\n",
                 (key >> 40) & 1 ? "GA_EM_BUILD_GRAD" : "GA_EM_BUILD_LOOKUP", ga_ctype(a), ga_ctype(o),
                 ga_ctype(i), a == GA_DOUBLE || o == GA_DOUBLE ? "ga_double" : "ga_float",
                 (unsigned)((key >> 24) & 0xff), (unsigned)((key >> 32) & 0xff),
                 (unsigned)((key >> 41) & 1), (unsigned)((key >> 48) & 0xff),
                 (key >> 56) ? (unsigned)((key >> 56) & 15) : 1u, (key >> 60) ? (unsigned)(key >> 60) : 1u);
}

static int check_types(gpucontext *ctx, const GpuArray *a, const GpuArray *o, const GpuArray *ids) {
  if (!is_real(a->typecode) || !is_real(o->typecode))
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR, "Rows must be half, float or double");
  if (!ga_lm_is_id(ids->typecode))
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR, "Token ids must be 32- or 64-bit integers");
  return GA_NO_ERROR;
}

/* `by_token`: out or dout; `by_row`: the table or dtable */
static int check_shapes(gpucontext *ctx, const GpuArray *by_token, const char *name,
                        const GpuArray *by_row, const GpuArray *ids) {
  if (by_row->nd != 2)
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "The table has %u dimensions, expected 2", by_row->nd);
  if (by_token->nd != ids->nd + 1 || !ga_lm_same_dims(by_token, ids, ids->nd) ||
      by_token->dimensions[ids->nd] != by_row->dimensions[1])
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR,
                      "%s must have the dimensions of the ids and then the table's row length", name);
  return GA_NO_ERROR;
}

/* Elements per access: the widest for which a load is at most 16 bytes and a store 32, the rows
 * hold a whole number of them and every row of both arrays starts on a boundary of one. */
static unsigned vector_width(const GpuArray *in, const GpuArray *out, size_t width) {
  const GpuArray *a[2];
  unsigned e, i, k;
  a[0] = in;
  a[1] = out;
  e = 16 / (unsigned)gpuarray_get_elsize(in->typecode);
  while (e * gpuarray_get_elsize(out->typecode) > 32) e /= 2;
  for (; e > 1; e /= 2) {
    int ok = width % e == 0;
    for (k = 0; k < 2 && ok; k++) {
      size_t es = gpuarray_get_elsize(a[k]->typecode), b = es * e;
      if (a[k]->strides[a[k]->nd - 1] != (ssize_t)es) ok = 0;
      if ((a[k]->data->ptr + a[k]->offset) % b != 0) ok = 0;
      for (i = 0; i + 1 < a[k]->nd; i++)
        if (a[k]->dimensions[i] > 1 && a[k]->strides[i] % (ssize_t)b != 0) ok = 0;
    }
    if (ok) break;
  }
  return e;
}

/* Vectors of a thread: 16 bytes of the array that is read. */
static unsigned vectors_of_thread(const GpuArray *in, unsigned e) {
  const unsigned b = (unsigned)gpuarray_get_elsize(in->typecode) * e;
  return b >= 16 ? 1 : 16 / b;
}

static int fill(gpucontext *ctx, em_layout *L, ga_lead *lead, const GpuArray *by_token,
                const GpuArray *by_row, const GpuArray *ids, double scale, ssize_t pad, int flags,
                unsigned e) {
  const ssize_t *str[2];
  long long out[2][GA_LM_MAXD];
  int err;
  memset(L, 0, sizeof(*L));
  str[0] = ids->strides;
  str[1] = by_token->strides;
  err = ga_lm_lead(ctx, ids->nd, ids->dimensions, 2, str, lead, out);
  if (err != GA_NO_ERROR) return err;
  L->n = lead->count;
  L->v = by_row->dimensions[0];
  L->nv = (unsigned)(by_row->dimensions[1] / e);
  L->has_pad = ISSET(flags, GA_EMBED_PAD);
  L->pad = pad;
  L->scale = scale;
  memcpy(L->dims, lead->dims, sizeof(L->dims));
  memcpy(L->i_str, out[0], sizeof(L->i_str));
  memcpy(L->t_str, out[1], sizeof(L->t_str));
  L->t_col = by_token->strides[by_token->nd - 1];
  L->v_row = by_row->strides[0];
  L->v_col = by_row->strides[1];
  return GA_NO_ERROR;
}

/* what both calls refuse before anything is enqueued */
static int check_call(gpucontext *ctx, const GpuArray *by_row, double scale, int flags, int allowed) {
  if (flags & ~allowed) return ga_err_fmt(ctx->err, GA_INVALID_ERROR, "Unknown flags 0x%x", flags);
  if (!isfinite((float)scale)) return ga_err_set(ctx->err, GA_VALUE_ERROR, "scale is not a finite float");
  if (by_row->dimensions[0] > 0x7fffffffUL || by_row->dimensions[1] > 0x7fffffffUL)
    return ga_err_set(ctx->err, GA_XLARGE_ERROR, "The table has more than 2^31 - 1 rows or columns");
  if (ISSET(flags, GA_EMBED_CHECK) && ga_lm_capturing(ctx))
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR,
                      "A checked call waits and cannot be captured into a graph");
  return GA_NO_ERROR;
}

#define EM_TOKENS 256 /* GA_EM_TOKENS of the template */
#define EM_MOST 64
#define EM_CTAS 12    /* CTAs of 256 threads for every SM, of which it holds 8 at once where halfs or floats move
                         in 16-byte vectors without widening (32 registers a thread), 4 to 6 otherwise */

int GpuArray_embed(GpuArray *out, const GpuArray *table, const GpuArray *ids, double scale,
                   ssize_t pad, int flags) {
  gpucontext *ctx;
  const ga_function *fn;
  em_layout L;
  ga_lead lead;
  CUdeviceptr p_out, p_table, p_ids, p_err;
  void *params[5];
  unsigned grid[3] = {1, 1, 1}, block[3], e, c;
  unsigned long long blocks;
  int err;

  if (out == NULL || out->data == NULL) return GA_INVALID_ERROR;
  ctx = GpuArray_context(out);
  if ((err = ga_lm_check(ctx, out, "out", 1)) != GA_NO_ERROR ||
      (err = ga_lm_check(ctx, table, "table", 0)) != GA_NO_ERROR ||
      (err = ga_lm_check(ctx, ids, "ids", 0)) != GA_NO_ERROR ||
      (err = check_types(ctx, table, out, ids)) != GA_NO_ERROR ||
      (err = check_shapes(ctx, out, "out", table, ids)) != GA_NO_ERROR ||
      (err = check_call(ctx, table, scale, flags, GA_EMBED_PAD | GA_EMBED_CHECK)) != GA_NO_ERROR)
    return err;
  e = vector_width(table, out, table->dimensions[1]);
  c = vectors_of_thread(table, e);
  err = fill(ctx, &L, &lead, out, table, ids, scale, pad, flags, e);
  if (err != GA_NO_ERROR || L.n == 0 || L.nv == 0) return err;
  err = ga_lm_kernel(ctx, "ga_embed",
                     (uint64_t)table->typecode | (uint64_t)out->typecode << 8 |
                         (uint64_t)ids->typecode << 16 | (uint64_t)e << 24 | (uint64_t)lead.nd << 32 |
                         (uint64_t)c << 48,
                     emit, &fn);
  if (err != GA_NO_ERROR) return err;
  ga_lm_geometry((L.nv + c - 1) / c, 256, block, &grid[1]);
  /* Tokens of a group: as many as leave a few groups for every SM, at most EM_TOKENS of a CTA */
  L.chunk = EM_TOKENS / block[1] < EM_MOST ? EM_TOKENS / block[1] : EM_MOST;
  while (L.chunk > 1 && (L.n + L.chunk - 1) / L.chunk * grid[1] < (unsigned long long)ctx->num_sms * EM_CTAS * block[1])
    L.chunk /= 2;
  blocks = (L.n + (unsigned long long)block[1] * L.chunk - 1) / (block[1] * L.chunk);
  if (blocks > 0x7fffffffULL || grid[1] > 65535)
    return ga_err_set(ctx->err, GA_XLARGE_ERROR, "Too many tokens or too long rows for one call");
  grid[0] = (unsigned)blocks;
  p_out = out->data->ptr + out->offset;
  p_table = table->data->ptr + table->offset;
  p_ids = ids->data->ptr + ids->offset;
  p_err = ISSET(flags, GA_EMBED_CHECK) ? ga_lm_err_word(ctx) : 0;
  params[0] = &L;
  params[1] = &p_out;
  params[2] = &p_table;
  params[3] = &p_ids;
  params[4] = &p_err;
  err = ga_launch(ctx, fn, grid, block, 0, params);
  if (err == GA_NO_ERROR && ISSET(flags, GA_EMBED_CHECK))
    err = ga_lm_err_take(ctx, "A token id is outside the table");
  return err;
}

int GpuEmbedGrad_new(GpuEmbedGrad **eg, gpucontext *ctx) {
  GpuEmbedGrad *r;
  if (eg == NULL) return GA_INVALID_ERROR;
  *eg = NULL;
  if (ctx == NULL) return ga_err_set(ga_global_err, GA_INVALID_ERROR, "GpuEmbedGrad_new: no context");
  r = calloc(1, sizeof(*r));
  if (r == NULL) return ga_err_sys(ctx->err, "calloc");
  r->ctx = ctx;
  ctx->refcnt++;
  *eg = r;
  return GA_NO_ERROR;
}

void GpuEmbedGrad_free(GpuEmbedGrad *eg) {
  gpucontext *ctx;
  if (eg == NULL) return;
  ctx = eg->ctx;
  ga_workspace_free(&eg->ws);
  free(eg);
  ga_ctx_unref(ctx);
}

/* constants of the template */
#define EG_STEP 8        /* a multiple of GA_EG_U */
#define EG_X 64          /* threads along the rows: four or more share the joining of a run */
#define EG_FEW 1024      /* GA_EG_FEW */
#define EG_TX 32         /* GA_EG_TX */
#define EG_BITS 9        /* GA_EG_BITS */
#define EG_THREADS 512   /* GA_EG_THREADS */
#define EG_ROUND 2048    /* GA_EG_ROUND */
#define EG_GROUP_THREADS 1024
#define EG_CHUNKS 16 /* chunks for every SM at most, where each takes a CTA to join */
#define EG_CLUSTER 8     /* CTAs of the one-launch sort: one where EG_ALONE rounds are enough */
#define EG_ALONE 2
#define EG_MAX_ROUNDS 2  /* of EG_ROUND tokens for each CTA of the cluster; more tokens are sorted
                            sooner by all SMs in several launches (65000: 29 us, one cluster 39) */
#define EG_SHARED (16 * 512 * 4 + 8 * 512 * 4 + 512 * 4 + 16 * 4) /* ga__eg_shared without `keys` */
#define EG_MAX_TILES 128 /* every sorting CTA reads all tiles' counts: 256 KiB at most */

static int launch_direct(GpuEmbedGrad *eg, em_layout *L, uint64_t key, unsigned c, CUdeviceptr *p_dt,
                         CUdeviceptr *p_do, CUdeviceptr *p_ids, CUdeviceptr *p_err) {
  gpucontext *ctx = eg->ctx;
  const ga_function *fn;
  void *params[5];
  unsigned grid[3] = {1, 1, 1}, block[3] = {1, 1, 1};
  unsigned long long ctas;
  int err = ga_lm_kernel(ctx, "ga_eg_direct", key, emit, &fn);
  if (err != GA_NO_ERROR) return err;
  while (block[0] < EG_TX && block[0] * c < L->nv) block[0] *= 2;
  block[1] = 256 / block[0];
  grid[1] = (L->nv + block[0] * c - 1) / (block[0] * c);
  if (grid[1] > 65535) return ga_err_set(ctx->err, GA_XLARGE_ERROR, "Too long rows for one call");
  /* the slices of all row ranges fill the device about once */
  ctas = (unsigned long long)ctx->num_sms * 8 / grid[1];
  if (ctas == 0) ctas = 1;
  L->chunk = (unsigned)((L->v + ctas - 1) / ctas);
  grid[0] = (unsigned)((L->v + L->chunk - 1) / L->chunk);
  params[0] = L;
  params[1] = p_dt;
  params[2] = p_do;
  params[3] = p_ids;
  params[4] = p_err;
  return ga_launch(ctx, fn, grid, block, 0, params);
}

/* Zeros for all rows of dtable, beside the launch before this one. */
static int launch_zeros(GpuEmbedGrad *eg, const em_layout *L, uint64_t key, CUdeviceptr *p_dt, unsigned e,
                        size_t es) {
  gpucontext *ctx = eg->ctx;
  const ga_function *fn;
  const unsigned long long row = (unsigned long long)L->nv * e * es;
  unsigned long long bytes = 0, ctas;
  void *params[3];
  unsigned grid[3] = {1, 1, 1}, block[3] = {EG_THREADS, 1, 1};
  int err = ga_lm_kernel(ctx, "ga_eg_zero", key, emit, &fn);
  if (err != GA_NO_ERROR) return err;
  if (L->v_col == (long long)es && (L->v_row == (long long)row || L->v == 1) && *p_dt % 16 == 0) {
    bytes = row * L->v;
    ctas = (bytes + EG_THREADS * 64 - 1) / (EG_THREADS * 64);
  } else {
    ctas = (L->v + EG_THREADS / 32 - 1) / (EG_THREADS / 32);
  }
  if (ctas > 0x7fffffffULL) return ga_err_set(ctx->err, GA_XLARGE_ERROR, "The table is too large");
  grid[0] = ctas ? (unsigned)ctas : 1;
  params[0] = (void *)L;
  params[1] = p_dt;
  params[2] = &bytes;
  return ga_launch(ctx, fn, grid, block, 0, params);
}

int GpuEmbedGrad_call(GpuEmbedGrad *eg, GpuArray *dtable, const GpuArray *dout, const GpuArray *ids,
                      double scale, ssize_t pad, int flags) {
  gpucontext *ctx;
  const ga_function *sort, *count, *scatter, *sum, *join;
  em_layout L;
  ga_lead lead;
  eg_sort S;
  CUdeviceptr p_dt, p_do, p_ids, p_err, p_counts, p_key[2], p_order[2], p_off, p_part;
  void *params[9];
  unsigned grid[3] = {1, 1, 1}, block[3], flat[3] = {EG_THREADS, 1, 1}, g1[3] = {1, 1, 1}, e, c, ny, bits, last, rounds = 1;
  unsigned long long groups;
  size_t fsize, list, cbytes, es;
  uint64_t key;
  int err, accumulate, one;

  if (eg == NULL) return GA_INVALID_ERROR;
  ctx = eg->ctx;
  if ((err = ga_lm_check(ctx, dtable, "dtable", 1)) != GA_NO_ERROR ||
      (err = ga_lm_check(ctx, dout, "dout", 0)) != GA_NO_ERROR ||
      (err = ga_lm_check(ctx, ids, "ids", 0)) != GA_NO_ERROR ||
      (err = check_types(ctx, dout, dtable, ids)) != GA_NO_ERROR ||
      (err = check_shapes(ctx, dout, "dout", dtable, ids)) != GA_NO_ERROR ||
      (err = check_call(ctx, dtable, scale, flags, GA_EMBED_PAD | GA_EMBED_CHECK | GA_EMBED_ACCUMULATE)) !=
          GA_NO_ERROR)
    return err;
  accumulate = ISSET(flags, GA_EMBED_ACCUMULATE);
  es = gpuarray_get_elsize(dtable->typecode);
  e = vector_width(dout, dtable, dtable->dimensions[1]);
  c = vectors_of_thread(dout, e);
  err = fill(ctx, &L, &lead, dout, dtable, ids, scale, pad, flags, e);
  if (err != GA_NO_ERROR) return err;
  if (L.n > 0x7fffffffULL)
    return ga_err_set(ctx->err, GA_XLARGE_ERROR, "More than 2^31 - 1 tokens in one call");
  /* without tokens there are zeros to write at most, for rows that there are */
  if (L.nv == 0 || (L.n == 0 && (accumulate || L.v == 0))) return GA_NO_ERROR;

  key = (uint64_t)dout->typecode | (uint64_t)dtable->typecode << 8 | (uint64_t)ids->typecode << 16 |
        (uint64_t)e << 24 | (uint64_t)lead.nd << 32 | (uint64_t)1 << 40 | (uint64_t)accumulate << 41 |
        (uint64_t)c << 48;
  p_dt = dtable->data->ptr + dtable->offset;
  p_do = dout->data->ptr + dout->offset;
  p_ids = ids->data->ptr + ids->offset;
  p_err = ISSET(flags, GA_EMBED_CHECK) ? ga_lm_err_word(ctx) : 0;

  if (L.n <= EG_FEW && L.v > 0) {
    err = launch_direct(eg, &L, key, c, &p_dt, &p_do, &p_ids, &p_err);
    if (err == GA_NO_ERROR && ISSET(flags, GA_EMBED_CHECK))
      err = ga_lm_err_take(ctx, "A token id is outside the table");
    return err;
  }

  if ((err = ga_lm_kernel(ctx, "ga_eg_sum", key, emit, &sum)) != GA_NO_ERROR ||
      (err = ga_lm_kernel(ctx, "ga_eg_join", key, emit, &join)) != GA_NO_ERROR)
    return err;

  ga_lm_geometry((L.nv + c - 1) / c, EG_X, block, &ny);
  if (ny > 65535) return ga_err_set(ctx->err, GA_XLARGE_ERROR, "Too long rows for one call");
  grid[1] = ny;
  /* Chunks: threads for half the device, which with EG_STEP loads of a thread in flight keep the
   * memory busy; more and shorter ones only leave more parts to join. None shorter than one step. */
  groups = (unsigned long long)ctx->num_sms * EG_GROUP_THREADS / ((unsigned long long)block[0] * ny);
  if (groups > (unsigned long long)ctx->num_sms * EG_CHUNKS && block[0] >= 32)
    groups = (unsigned long long)ctx->num_sms * EG_CHUNKS;
  if (groups == 0) groups = 1;
  L.chunk = (unsigned)((L.n + groups - 1) / groups);
  L.chunk = (L.chunk + EG_STEP - 1) / EG_STEP * EG_STEP;
  L.chunks = (unsigned)((L.n + L.chunk - 1) / L.chunk);

  S.n = (unsigned)L.n;
  for (bits = 1; bits < 32 && (L.v >> bits) != 0; bits++) {} /* keys go up to V */
  S.passes = (bits + EG_BITS - 1) / EG_BITS;
  S.pass = 0;
  one = L.n <= (unsigned long long)EG_CLUSTER * EG_ROUND * EG_MAX_ROUNDS;
  if (one) {
    S.tiles = L.n <= EG_ROUND * EG_ALONE ? 1 : EG_CLUSTER;
    for (rounds = 1; (unsigned long long)S.tiles * EG_ROUND * rounds < L.n; rounds *= 2) {}
    S.tile = EG_ROUND * rounds;
  } else {
    S.tiles = (unsigned)((L.n + EG_ROUND - 1) / EG_ROUND);
    if (S.tiles > EG_MAX_TILES) S.tiles = EG_MAX_TILES;
    S.tile = (unsigned)(((L.n + S.tiles - 1) / S.tiles + EG_ROUND - 1) / EG_ROUND * EG_ROUND);
    S.tiles = (unsigned)((L.n + S.tile - 1) / S.tile);
  }

  fsize = dout->typecode == GA_DOUBLE || dtable->typecode == GA_DOUBLE ? 8 : 4;
  list = ((size_t)(L.n + EG_STEP) * 4 + 511) / 512 * 512;
  cbytes = one ? 0 : (size_t)EG_THREADS * S.tiles * 4;
  /* the sorted keys and offsets; for many tokens the counts and the lists between the passes */
  err = ga_workspace_need(ctx, &eg->ws, 3 * list + (one ? 0 : cbytes + 3 * list) +
                                            2 * (size_t)L.chunks * ny * block[0] * c * e * fsize);
  if (err != GA_NO_ERROR) return err;
  p_key[0] = eg->ws.cur->ptr;
  p_off = p_key[0] + list;
  p_part = p_off + 2 * list;
  if (!one) {
    p_key[1] = p_part;
    p_order[0] = p_key[1] + list;
    p_order[1] = p_order[0] + list;
    p_counts = p_order[1] + list;
    p_part = p_counts + cbytes;
  }

  params[0] = &L;
  params[1] = &S;
  g1[0] = S.tiles;
  if (one) {
    if ((err = ga_lm_kernel(ctx, "ga_eg_sort_all", key | (uint64_t)rounds << 56 | (uint64_t)S.tiles << 60, emit,
                            &sort)) != GA_NO_ERROR)
      return err;
    params[2] = &p_ids;
    params[3] = &p_key[0];
    params[4] = &p_off;
    params[5] = &p_err;
    last = 0;
    err = ga_launch(ctx, sort, g1, flat, EG_SHARED + (size_t)S.tile * 8, params);
  } else {
    if ((err = ga_lm_kernel(ctx, "ga_eg_count", key, emit, &count)) != GA_NO_ERROR ||
        (err = ga_lm_kernel(ctx, "ga_eg_scatter", key, emit, &scatter)) != GA_NO_ERROR)
      return err;
    last = (S.passes - 1) % 2;
    params[2] = &p_counts;
    params[3] = &p_ids;
    for (; S.pass < S.passes && err == GA_NO_ERROR; S.pass++) {
      params[4] = &p_key[1 - S.pass % 2];
      params[5] = &p_err;
      err = ga_launch(ctx, count, g1, flat, 0, params);
      if (err != GA_NO_ERROR) break;
      params[5] = &p_order[1 - S.pass % 2];
      params[6] = &p_key[S.pass % 2];
      params[7] = &p_order[S.pass % 2];
      params[8] = &p_off;
      err = ga_launch(ctx, scatter, g1, flat, 0, params);
    }
  }
  if (err == GA_NO_ERROR && !accumulate && L.v > 0) err = launch_zeros(eg, &L, key, &p_dt, e, es);

  if (err == GA_NO_ERROR) {
    grid[0] = (L.chunks + block[1] - 1) / block[1];
    params[1] = &p_dt;
    params[2] = &p_do;
    params[3] = &p_key[last];
    params[4] = &p_off;
    params[5] = &p_part;
    err = ga_launch(ctx, sum, grid, block, 0, params);
  }
  if (err == GA_NO_ERROR && L.chunks > 1) {
    params[2] = &p_key[last];
    params[3] = &p_part;
    grid[0] = block[0] < 32 ? (L.chunks + 6) / 8 : L.chunks - 1;
    err = ga_launch(ctx, join, grid, block, 0, params);
  }
  if (err == GA_NO_ERROR && ISSET(flags, GA_EMBED_CHECK))
    err = ga_lm_err_take(ctx, "A token id is outside the table");
  return err;
}
