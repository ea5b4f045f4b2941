/* The norm over a list of arrays, and clipping by it
 * (include/gpuarray/clipnorm.h; kernels in templates/ga_clipnorm.cuh). */
#include <math.h>
#include "private.h"

#define CN_MAX_CAP 960     /* entries of the largest table: a parameter block holds 32764 bytes */
#define CN_VECS 2048       /* GA_CN_VECS of the template */
#define CN_CTAS_PER_SM 8   /* 256 threads each; an SM holds 5 of them at once (48 registers a thread) */

typedef struct cn_item { /* the template's ga__cn_item */
  CUdeviceptr src, dst;
  unsigned long long n;
  unsigned int first;
  short stype, dtype;
} cn_item;

typedef struct cn_layout { /* the template's ga__cn_layout */
  unsigned int count, blocks, slot, slots;
  double scale, limit;
  cn_item item[CN_MAX_CAP];
} cn_layout;

#define CN_RESULT_BYTES 64 /* the template's ga__cn_result, then the partials */

struct _GpuClipNorm {
  gpucontext *ctx;
  unsigned int ctas;       /* of the largest launch */
  unsigned int launches;   /* at most */
  gpudata *mem;            /* result, partials[launches * ctas] */
  cn_layout *table;        /* filled anew by every call */
  struct cn_span *span;    /* for the overlap check */
  unsigned int nspan;
};

typedef struct cn_span {
  unsigned long long lo, hi;
  unsigned int at; /* index * 2 + (1: destination) */
} cn_span;

static void emit(ga_strb *sb, uint64_t key) {
  ga_strb_printf(sb, "#include \"cluda.h\"\n#define GA_CN_CAP %u\n#include \"ga_clipnorm.cuh\"\n",
                 (unsigned)key);
}

int GpuClipNorm_new(GpuClipNorm **cn, gpucontext *ctx) {
  GpuClipNorm *r;
  size_t bytes;
  int err = GA_NO_ERROR;
  if (cn == NULL) return GA_INVALID_ERROR;
  *cn = NULL;
  if (ctx == NULL) return ga_err_set(ga_global_err, GA_INVALID_ERROR, "GpuClipNorm_new: no context");
  r = calloc(1, sizeof(*r));
  if (r != NULL) r->table = calloc(1, sizeof(*r->table));
  if (r == NULL || r->table == NULL) {
    free(r);
    return ga_err_sys(ctx->err, "calloc");
  }
  r->ctas = ctx->num_sms * CN_CTAS_PER_SM;
  r->launches = (GA_CLIPNORM_MAX_ARRAYS + CN_MAX_CAP - 1) / CN_MAX_CAP;
  bytes = CN_RESULT_BYTES + (size_t)r->launches * r->ctas * sizeof(double);
  r->mem = gpudata_alloc(ctx, bytes, NULL, 0, &err);
  if (r->mem != NULL) err = gpudata_memset(r->mem, 0, 0); /* the ticket starts at zero */
  if (err != GA_NO_ERROR) {
    if (r->mem != NULL) gpudata_release(r->mem);
    free(r->table);
    free(r);
    return err;
  }
  r->ctx = ctx;
  ctx->refcnt++;
  *cn = r;
  return GA_NO_ERROR;
}

void GpuClipNorm_free(GpuClipNorm *cn) {
  gpucontext *ctx;
  if (cn == NULL) return;
  ctx = cn->ctx;
  gpudata_release(cn->mem);
  free(cn->table);
  free(cn->span);
  free(cn);
  ga_ctx_unref(ctx);
}

static int type_index(int tc) { return tc == GA_HALF ? 0 : tc == GA_FLOAT ? 1 : tc == GA_DOUBLE ? 2 : -1; }

static unsigned long long elements(const GpuArray *a) {
  unsigned long long n = 1;
  unsigned int i;
  for (i = 0; i < a->nd; i++) n *= a->dimensions[i];
  return n;
}

static int by_start(const void *a, const void *b) {
  const cn_span *x = a, *y = b;
  if (x->lo != y->lo) return x->lo < y->lo ? -1 : 1;
  return x->at < y->at ? -1 : x->at > y->at;
}

/* Sources may overlap each other; a destination (the norm too, as array n) may overlap nothing but
 * be its own source. */
static int check_overlap(GpuClipNorm *cn, const GpuArray *norm, GpuArray *const *dst,
                         const GpuArray *const *src, unsigned int n) {
  unsigned int i, k = 0;
  int sorted = 1;
  unsigned long long reach_dst = 0, reach_any = 0; /* ends of what came before */
  unsigned int who_any = 0, who_dst = 0;
  if (2 * (size_t)n + 1 > cn->nspan) {
    cn_span *s = realloc(cn->span, (2 * (size_t)n + 1) * sizeof(*s));
    if (s == NULL) return ga_err_sys(cn->ctx->err, "realloc");
    cn->span = s;
    cn->nspan = 2 * n + 1;
  }
  for (i = 0; i < n; i++) {
    const unsigned long long cnt = elements(src[i]);
    const unsigned long long s = src[i]->data->ptr + src[i]->offset, d = dst[i]->data->ptr + dst[i]->offset;
    if (cnt == 0) continue;
    cn->span[k].lo = d;
    cn->span[k].hi = d + cnt * gpuarray_get_elsize(dst[i]->typecode);
    cn->span[k].at = 2 * i + 1;
    if (k > 0 && d < cn->span[k - 1].lo) sorted = 0;
    k++;
    if (s == d && src[i]->typecode == dst[i]->typecode) continue; /* in place */
    cn->span[k].lo = s;
    cn->span[k].hi = s + cnt * gpuarray_get_elsize(src[i]->typecode);
    cn->span[k].at = 2 * i;
    if (s < d) sorted = 0;
    k++;
  }
  cn->span[k].lo = norm->data->ptr + norm->offset;
  cn->span[k].hi = cn->span[k].lo + gpuarray_get_elsize(norm->typecode);
  cn->span[k].at = 2 * n + 1;
  if (k > 0 && cn->span[k].lo < cn->span[k - 1].lo) sorted = 0;
  k++;
  if (!sorted) qsort(cn->span, k, sizeof(*cn->span), by_start);
  for (i = 0; i < k; i++) {
    const cn_span *p = &cn->span[i];
    const int is_dst = (int)(p->at & 1);
    const unsigned long long reach = is_dst ? reach_any : reach_dst;
    if (p->lo < reach)
      return ga_err_fmt(cn->ctx->err, GA_VALUE_ERROR,
                        "Array %u overlaps array %u and one of them is a destination", p->at / 2,
                        (is_dst ? who_any : who_dst) / 2);
    if (p->hi > reach_any) reach_any = p->hi, who_any = p->at;
    if (is_dst && p->hi > reach_dst) reach_dst = p->hi, who_dst = p->at;
  }
  return GA_NO_ERROR;
}

/* The same where the norm is the only destination. */
static int check_norm_overlap(gpucontext *ctx, const GpuArray *norm, const GpuArray *const *src, unsigned int n) {
  const unsigned long long lo = norm->data->ptr + norm->offset, hi = lo + gpuarray_get_elsize(norm->typecode);
  unsigned int i;
  for (i = 0; i < n; i++) {
    const unsigned long long cnt = elements(src[i]), s = src[i]->data->ptr + src[i]->offset;
    if (cnt > 0 && s < hi && lo < s + cnt * gpuarray_get_elsize(src[i]->typecode))
      return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "The norm overlaps src[%u]", i);
  }
  return GA_NO_ERROR;
}

/* ga_lm_check, the array's place in the list named only where there is something to say */
static int check_listed(gpucontext *ctx, const GpuArray *a, const char *list, unsigned int i, int dest) {
  char why[GA_ERR_MSGLEN];
  const int err = ga_lm_check(ctx, a, "the array", dest);
  if (err == GA_NO_ERROR) return err;
  memcpy(why, ctx->err->msg, sizeof(why));
  return ga_err_fmt(ctx->err, err, "%s[%u]: %.900s", list, i, why);
}

static int check_one(gpucontext *ctx, const GpuArray *s, const GpuArray *d, unsigned int i) {
  int err, f = GA_C_CONTIGUOUS | GA_F_CONTIGUOUS;
  if ((err = check_listed(ctx, s, "src", i, 0)) != GA_NO_ERROR) return err;
  if (type_index(s->typecode) < 0)
    return ga_err_fmt(ctx->err, GA_UNSUPPORTED_ERROR, "src[%u] must be half, float or double", i);
  if (!(s->flags & f))
    return ga_err_fmt(ctx->err, GA_INVALID_ERROR, "src[%u] is not one segment of memory", i);
  if (d == NULL || d == s) return d == NULL ? GA_NO_ERROR : check_listed(ctx, d, "dst", i, 1);
  if ((err = check_listed(ctx, d, "dst", i, 1)) != GA_NO_ERROR) return err;
  if (d->typecode != s->typecode && !(s->typecode == GA_HALF && d->typecode == GA_FLOAT))
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "dst[%u] must have the type of src[%u], or be float for half",
                      i, i);
  if (d->nd != s->nd || !ga_lm_same_dims(s, d, s->nd))
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "dst[%u] has not the shape of src[%u]", i, i);
  if (!(s->flags & d->flags & f))
    return ga_err_fmt(ctx->err, GA_INVALID_ERROR, "dst[%u] has not the order of src[%u] in memory", i, i);
  return GA_NO_ERROR;
}

/* Fills the table with arrays from *at on, as many as fit; *at moves on. */
static int fill(GpuClipNorm *cn, GpuArray *const *dst, const GpuArray *const *src, unsigned int n,
                unsigned int *at) {
  cn_layout *L = cn->table;
  unsigned long long blocks = 0;
  L->count = 0;
  for (; *at < n && L->count < CN_MAX_CAP; (*at)++) {
    const GpuArray *s = src[*at];
    const size_t es = gpuarray_get_elsize(s->typecode);
    cn_item *t = &L->item[L->count];
    t->n = elements(s);
    if (t->n == 0) continue;
    t->src = s->data->ptr + s->offset;
    t->dst = dst != NULL ? dst[*at]->data->ptr + dst[*at]->offset : 0;
    t->stype = (short)type_index(s->typecode);
    t->dtype = dst != NULL ? (short)type_index(dst[*at]->typecode) : t->stype;
    t->first = (unsigned)blocks;
    /* vectors from the 16-byte boundary at or below the first element */
    blocks += ((t->n * es + (t->src & 15) + 15) / 16 + CN_VECS - 1) / CN_VECS;
    if (blocks > 0x7fffffffULL)
      return ga_err_set(cn->ctx->err, GA_XLARGE_ERROR, "The arrays are too large for one call");
    L->count++;
  }
  L->blocks = (unsigned)blocks;
  return GA_NO_ERROR;
}

int GpuClipNorm_call(GpuClipNorm *cn, GpuArray *norm, GpuArray *const *dst,
                     const GpuArray *const *src, unsigned int n, double scale, double limit) {
  gpucontext *ctx;
  const ga_function *fn, *fs;
  cn_layout *L;
  CUdeviceptr p_part, p_res, p_norm;
  void *params[5];
  unsigned grid[3] = {1, 1, 1}, block[3] = {256, 1, 1}, i, at, cap;
  int err, is_double;

  if (cn == NULL) return GA_INVALID_ERROR;
  ctx = cn->ctx;
  L = cn->table;
  if ((err = ga_lm_check(ctx, norm, "norm", 1)) != GA_NO_ERROR) return err;
  if (norm->nd != 0 || (norm->typecode != GA_FLOAT && norm->typecode != GA_DOUBLE))
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "norm must be 0-d, float or double");
  if (n > 0 && src == NULL) return ga_err_set(ctx->err, GA_INVALID_ERROR, "src is missing");
  if (n > GA_CLIPNORM_MAX_ARRAYS)
    return ga_err_fmt(ctx->err, GA_XLARGE_ERROR, "More than %d arrays", GA_CLIPNORM_MAX_ARRAYS);
  if (!isfinite(scale) || !(limit >= 0))
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "scale must be finite, limit 0 or more");
  for (i = 0; i < n; i++) {
    if (dst != NULL && dst[i] == NULL)
      return ga_err_fmt(ctx->err, GA_INVALID_ERROR, "dst[%u] is missing", i);
    err = check_one(ctx, src[i], dst != NULL ? dst[i] : NULL, i);
    if (err != GA_NO_ERROR) return err;
  }
  err = dst != NULL ? check_overlap(cn, norm, dst, src, n) : check_norm_overlap(ctx, norm, src, n);
  if (err != GA_NO_ERROR) return err;

  /* the smallest table that holds the list: what a launch carries is copied with it */
  cap = n <= 32 ? 32 : n <= 128 ? 128 : CN_MAX_CAP;
  if ((err = ga_lm_kernel(ctx, "ga_cn_norm", cap, emit, &fn)) != GA_NO_ERROR ||
      (err = ga_lm_kernel(ctx, "ga_cn_scale", cap, emit, &fs)) != GA_NO_ERROR)
    return err;
  L->scale = scale;
  L->limit = limit;
  p_res = cn->mem->ptr;
  p_part = p_res + CN_RESULT_BYTES;
  p_norm = norm->data->ptr + norm->offset;
  is_double = norm->typecode == GA_DOUBLE;

  params[0] = L;
  params[1] = &p_part;
  params[2] = &p_res;
  params[3] = &p_norm;
  params[4] = &is_double;
  at = 0;
  L->slot = 0;
  do {
    err = fill(cn, dst, src, n, &at);
    if (err != GA_NO_ERROR) return err;
    grid[0] = L->blocks < cn->ctas ? (L->blocks ? L->blocks : 1) : cn->ctas;
    L->slots = at == n ? L->slot + grid[0] : 0;
    err = ga_launch(ctx, fn, grid, block, 0, params);
    if (err != GA_NO_ERROR) return err;
    L->slot += grid[0];
  } while (at < n);
  if (dst == NULL) return GA_NO_ERROR;

  params[1] = &p_res;
  for (at = 0; at < n;) {
    /* a list of one table is still in place */
    if (n > CN_MAX_CAP) {
      err = fill(cn, dst, src, n, &at);
      if (err != GA_NO_ERROR) return err;
    } else {
      at = n;
    }
    if (L->blocks == 0) continue;
    grid[0] = L->blocks;
    err = ga_launch(ctx, fs, grid, block, 0, params);
    if (err != GA_NO_ERROR) return err;
  }
  return GA_NO_ERROR;
}
