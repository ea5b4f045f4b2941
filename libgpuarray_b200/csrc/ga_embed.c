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

typedef struct eg_fill { /* the templates' ga__eg_fill */
  CUdeviceptr p;
  unsigned long long bytes, r0, r1;
} eg_fill;

typedef struct eg_sort { /* the templates' ga__eg_sort */
  unsigned int n, tiles, tile, passes, pass;
} eg_sort;

struct _GpuEmbedGrad {
  gpucontext *ctx;
  ga_workspace ws;
};

static int is_real(int tc) { return tc == GA_HALF || tc == GA_FLOAT || tc == GA_DOUBLE; }

/* key: A type | O type << 8 | id type << 16 | E << 24 | ND << 32 | gradient << 40 | accumulate << 41 */
static void emit(ga_strb *sb, uint64_t key) {
  const int a = (int)(key & 0xff), o = (int)((key >> 8) & 0xff), i = (int)((key >> 16) & 0xff);
  ga_strb_printf(sb,
                 "#include \"cluda.h\"\n#define %s\n#define GA_EM_A_T %s\n#define GA_EM_O_T %s\n"
                 "#define GA_EM_I_T %s\n#define GA_EM_F_T %s\n#define GA_EM_E %u\n"
                 "#define GA_EM_ND %u\n#define GA_EM_ACCUMULATE %u\n#include \"ga_embed.cuh\"\n",
                 (key >> 40) & 1 ? "GA_EM_BUILD_GRAD" : "GA_EM_BUILD_LOOKUP", ga_ctype(a), ga_ctype(o),
                 ga_ctype(i), a == GA_DOUBLE || o == GA_DOUBLE ? "ga_double" : "ga_float",
                 (unsigned)((key >> 24) & 0xff), (unsigned)((key >> 32) & 0xff),
                 (unsigned)((key >> 41) & 1));
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
#define EM_CTAS 6     /* CTAs of 256 threads for every SM */

int GpuArray_embed(GpuArray *out, const GpuArray *table, const GpuArray *ids, double scale,
                   ssize_t pad, int flags) {
  gpucontext *ctx;
  const ga_function *fn;
  em_layout L;
  ga_lead lead;
  CUdeviceptr p_out, p_table, p_ids, p_err;
  void *params[5];
  unsigned grid[3] = {1, 1, 1}, block[3], e;
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
  err = fill(ctx, &L, &lead, out, table, ids, scale, pad, flags, e);
  if (err != GA_NO_ERROR || L.n == 0 || L.nv == 0) return err;
  err = ga_lm_kernel(ctx, "ga_embed",
                     (uint64_t)table->typecode | (uint64_t)out->typecode << 8 |
                         (uint64_t)ids->typecode << 16 | (uint64_t)e << 24 | (uint64_t)lead.nd << 32,
                     emit, &fn);
  if (err != GA_NO_ERROR) return err;
  ga_lm_geometry(L.nv, block, &grid[1]);
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
#define EG_STEP 8        /* GA_EG_U */
#define EG_FEW 512       /* GA_EG_FEW */
#define EG_TX 32         /* GA_EG_TX */
#define EG_BITS 9        /* GA_EG_BITS */
#define EG_THREADS 512   /* GA_EG_THREADS */
#define EG_ROUND 2048    /* GA_EG_ROUND */
#define EG_GROUP_THREADS 1024
#define EG_MAX_TILES 128 /* every sorting CTA reads all tiles' counts: 256 KiB at most */

static int launch_direct(GpuEmbedGrad *eg, em_layout *L, uint64_t key, CUdeviceptr *p_dt,
                         CUdeviceptr *p_do, CUdeviceptr *p_ids, CUdeviceptr *p_err) {
  gpucontext *ctx = eg->ctx;
  const ga_function *fn;
  void *params[5];
  unsigned grid[3] = {1, 1, 1}, block[3] = {1, 1, 1};
  unsigned long long ctas;
  int err = ga_lm_kernel(ctx, "ga_eg_direct", key, emit, &fn);
  if (err != GA_NO_ERROR) return err;
  while (block[0] < EG_TX && block[0] < L->nv) block[0] *= 2;
  block[1] = 256 / block[0];
  grid[1] = (L->nv + block[0] - 1) / block[0];
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

/* The part `i` of `parts` of dtable's rows for the CTAs beside a sorting launch to write zeros to. */
static void fill_part(eg_fill *F, const em_layout *L, CUdeviceptr p_dt, unsigned e, size_t es,
                      int accumulate, unsigned i, unsigned parts) {
  const unsigned long long row = (unsigned long long)L->nv * e * es, all = row * L->v;
  memset(F, 0, sizeof(*F));
  F->p = p_dt;
  if (accumulate) return;
  if (L->v_col == (long long)es && (L->v_row == (long long)row || L->v == 1) && p_dt % 16 == 0) {
    const unsigned long long step = (all / parts + 15) / 16 * 16, lo = step * i < all ? step * i : all;
    F->p = p_dt + lo;
    F->bytes = i + 1 == parts || all - lo < step ? all - lo : step;
  } else {
    F->r0 = L->v * i / parts;
    F->r1 = L->v * (i + 1) / parts;
  }
}

int GpuEmbedGrad_call(GpuEmbedGrad *eg, GpuArray *dtable, const GpuArray *dout, const GpuArray *ids,
                      double scale, ssize_t pad, int flags) {
  gpucontext *ctx;
  const ga_function *count, *scatter, *sum, *join;
  em_layout L;
  ga_lead lead;
  eg_fill F;
  eg_sort S;
  CUdeviceptr p_dt, p_do, p_ids, p_err, p_counts, p_key[2], p_order[2], p_off, p_part;
  void *params[10];
  unsigned grid[3] = {1, 1, 1}, block[3], flat[3] = {EG_THREADS, 1, 1}, g1[3] = {1, 1, 1}, e, ny, bits, last;
  unsigned long long groups;
  size_t fsize, list, cbytes, es;
  uint64_t key;
  int err, accumulate;

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
  err = fill(ctx, &L, &lead, dout, dtable, ids, scale, pad, flags, e);
  if (err != GA_NO_ERROR) return err;
  if (L.n > 0x7fffffffULL)
    return ga_err_set(ctx->err, GA_XLARGE_ERROR, "More than 2^31 - 1 tokens in one call");
  if (L.nv == 0 || (L.n == 0 && accumulate)) return GA_NO_ERROR;

  key = (uint64_t)dout->typecode | (uint64_t)dtable->typecode << 8 | (uint64_t)ids->typecode << 16 |
        (uint64_t)e << 24 | (uint64_t)lead.nd << 32 | (uint64_t)1 << 40 | (uint64_t)accumulate << 41;
  p_dt = dtable->data->ptr + dtable->offset;
  p_do = dout->data->ptr + dout->offset;
  p_ids = ids->data->ptr + ids->offset;
  p_err = ISSET(flags, GA_EMBED_CHECK) ? ga_lm_err_word(ctx) : 0;

  if (L.n <= EG_FEW && L.v > 0) {
    err = launch_direct(eg, &L, key, &p_dt, &p_do, &p_ids, &p_err);
    if (err == GA_NO_ERROR && ISSET(flags, GA_EMBED_CHECK))
      err = ga_lm_err_take(ctx, "A token id is outside the table");
    return err;
  }

  if ((err = ga_lm_kernel(ctx, "ga_eg_count", key, emit, &count)) != GA_NO_ERROR ||
      (err = ga_lm_kernel(ctx, "ga_eg_scatter", key, emit, &scatter)) != GA_NO_ERROR ||
      (err = ga_lm_kernel(ctx, "ga_eg_sum", key, emit, &sum)) != GA_NO_ERROR ||
      (err = ga_lm_kernel(ctx, "ga_eg_join", key, emit, &join)) != GA_NO_ERROR)
    return err;

  ga_lm_geometry(L.nv, block, &ny);
  if (ny > 65535) return ga_err_set(ctx->err, GA_XLARGE_ERROR, "Too long rows for one call");
  grid[1] = ny;
  /* Chunks: threads for half the device, which with EG_STEP loads of a thread in flight keep the
   * memory busy; more and shorter ones only leave more parts to join. None shorter than one step. */
  groups = (unsigned long long)ctx->num_sms * EG_GROUP_THREADS / ((unsigned long long)block[0] * ny);
  if (groups == 0) groups = 1;
  L.chunk = (unsigned)((L.n + groups - 1) / groups);
  L.chunk = (L.chunk + EG_STEP - 1) / EG_STEP * EG_STEP;
  L.chunks = (unsigned)((L.n + L.chunk - 1) / L.chunk);

  S.n = (unsigned)L.n;
  S.tiles = (unsigned)((L.n + EG_ROUND - 1) / EG_ROUND);
  if (S.tiles > EG_MAX_TILES) S.tiles = EG_MAX_TILES;
  S.tile = (unsigned)(((L.n + S.tiles - 1) / S.tiles + EG_ROUND - 1) / EG_ROUND * EG_ROUND);
  S.tiles = (unsigned)((L.n + S.tile - 1) / S.tile);
  for (bits = 1; bits < 32 && (L.v >> bits) != 0; bits++) {} /* keys go up to V */
  S.passes = (bits + EG_BITS - 1) / EG_BITS;

  fsize = dout->typecode == GA_DOUBLE || dtable->typecode == GA_DOUBLE ? 8 : 4;
  list = ((size_t)(L.n + EG_STEP) * 4 + 511) / 512 * 512;
  cbytes = (size_t)S.passes * EG_THREADS * S.tiles * 4;
  err = ga_workspace_need(ctx, &eg->ws, cbytes + 6 * list + 2 * (size_t)L.chunks * L.nv * e * fsize);
  if (err != GA_NO_ERROR) return err;
  p_counts = eg->ws.cur->ptr;
  p_key[0] = p_counts + cbytes;
  p_order[0] = p_key[0] + list;
  p_key[1] = p_order[0] + list;
  p_order[1] = p_key[1] + list;
  p_off = p_order[1] + list;
  p_part = p_off + 2 * list;

  /* the CTAs that write zeros: what the device holds beside the sorting ones */
  g1[0] = S.tiles + (accumulate ? 0 : ctx->num_sms * 4 > S.tiles + ctx->num_sms ? ctx->num_sms * 4 - S.tiles : ctx->num_sms);
  params[0] = &L;
  params[1] = &S;
  params[2] = &F;
  params[3] = &p_counts;
  params[4] = &p_ids;
  params[5] = &p_err;
  fill_part(&F, &L, p_dt, e, es, accumulate, 0, S.passes + 1);
  err = ga_launch(ctx, count, g1, flat, 0, params);
  for (S.pass = 0; S.pass < S.passes && err == GA_NO_ERROR; S.pass++) {
    fill_part(&F, &L, p_dt, e, es, accumulate, S.pass + 1, S.passes + 1);
    params[5] = &p_key[1 - S.pass % 2];
    params[6] = &p_order[1 - S.pass % 2];
    params[7] = &p_key[S.pass % 2];
    params[8] = &p_order[S.pass % 2];
    params[9] = &p_off;
    err = ga_launch(ctx, scatter, g1, flat, 0, params);
  }
  last = (S.passes - 1) % 2;

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
    err = ga_launch(ctx, join, grid, block, 0, params);
  }
  if (err == GA_NO_ERROR && ISSET(flags, GA_EMBED_CHECK))
    err = ga_lm_err_take(ctx, "A token id is outside the table");
  return err;
}
