/* What the language-model operators (ga_embed.c, ga_logprobs.c, ga_clipnorm.c)
 * share on the host: argument checks, collapsing of the dimensions that index
 * tokens or rows, compiled kernels, workspaces, the error word. */
#include "private.h"

int ga_lm_is_id(int typecode) {
  return typecode == GA_INT || typecode == GA_UINT || typecode == GA_LONG || typecode == GA_ULONG;
}

int ga_lm_check(gpucontext *ctx, const GpuArray *a, const char *what, int dest) {
  unsigned int i;
  if (a == NULL || a->data == NULL)
    return ga_err_fmt(ctx->err, GA_INVALID_ERROR, "%s is missing", what);
  if (GpuArray_context(a) != ctx)
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "%s belongs to another context", what);
  if (dest && !GpuArray_ISWRITEABLE(a))
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "%s is not writeable", what);
  /* the flag speaks of the offset and the strides; a wrapped buffer may itself start anywhere */
  if (!GpuArray_ISALIGNED(a) || (a->data->ptr + a->offset) % gpuarray_get_elsize(a->typecode) != 0)
    return ga_err_fmt(ctx->err, GA_UNALIGNED_ERROR, "%s is not aligned", what);
  if (!ga_array_in_bounds(a))
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "%s reaches outside its buffer", what);
  for (i = 0; i < a->nd; i++)
    if (a->dimensions[i] == 0) return GA_NO_ERROR;
  if (dest)
    for (i = 0; i < a->nd; i++)
      if (a->dimensions[i] > 1 && a->strides[i] == 0)
        return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "%s has a stride of 0 in dimension %u", what, i);
  return GA_NO_ERROR;
}

int ga_lm_same_dims(const GpuArray *a, const GpuArray *b, unsigned int nd) {
  unsigned int i;
  for (i = 0; i < nd; i++)
    if (a->dimensions[i] != b->dimensions[i]) return 0;
  return 1;
}

#define LM_MAXND 16
#define LM_MAXARR 8

int ga_lm_lead(gpucontext *ctx, unsigned int nd, const size_t *dims, unsigned int n,
               const ssize_t *const *str, ga_lead *lead, long long (*out)[GA_LM_MAXD]) {
  size_t d[LM_MAXND];
  ssize_t s[LM_MAXARR][LM_MAXND], *ps[LM_MAXARR];
  unsigned int i, k;
  memset(lead, 0, sizeof(*lead));
  lead->nd = 1;
  lead->count = 1;
  lead->dims[0] = 1;
  for (k = 0; k < n; k++) memset(out[k], 0, sizeof(out[k]));
  if (nd > LM_MAXND || n > LM_MAXARR)
    return ga_err_fmt(ctx->err, GA_UNSUPPORTED_ERROR, "More than %d dimensions", LM_MAXND);
  for (i = 0; i < nd; i++) {
    d[i] = dims[i];
    lead->count *= dims[i];
  }
  if (nd == 0 || lead->count == 0) return GA_NO_ERROR;
  for (k = 0; k < n; k++) {
    ps[k] = NULL;
    if (str[k] == NULL) continue;
    memcpy(s[k], str[k], nd * sizeof(ssize_t));
    ps[k] = s[k];
  }
  gpuarray_elemwise_collapse(n, &nd, d, ps);
  if (nd > GA_LM_MAXD)
    return ga_err_fmt(ctx->err, GA_UNSUPPORTED_ERROR,
                      "More than %d dimensions remain after collapsing", GA_LM_MAXD);
  lead->nd = nd;
  for (i = 0; i < nd; i++) {
    lead->dims[i] = d[i];
    for (k = 0; k < n; k++)
      if (ps[k] != NULL) out[k][i] = s[k][i];
  }
  return GA_NO_ERROR;
}

/* ------------------------------------------------------------------ kernels */

typedef struct lm_entry {
  const char *fname; /* compared by its text */
  uint64_t key;
  ga_function fn;
  struct lm_entry *next;
} lm_entry;

int ga_lm_kernel(gpucontext *ctx, const char *fname, uint64_t key,
                 void (*emit)(ga_strb *sb, uint64_t key), const ga_function **fn) {
  lm_entry *e;
  ga_strb sb;
  ga_function got;
  int err;
  for (e = (lm_entry *)ctx->lm_cache; e != NULL; e = e->next)
    if (e->key == key && (e->fname == fname || strcmp(e->fname, fname) == 0)) {
      *fn = &e->fn;
      return GA_NO_ERROR;
    }
  ga_strb_init(&sb);
  emit(&sb, key);
  if (sb.failed) {
    ga_strb_free(&sb);
    return ga_err_set(ctx->err, GA_MEMORY_ERROR, "Out of memory");
  }
  err = ga_compile(ctx, ga_strb_cstr(&sb), fname, NULL, &got, NULL);
  ga_strb_free(&sb);
  if (err != GA_NO_ERROR) return err;
  got.dependent_ok = 1; /* the templates begin with ga__grid_dependency_sync() */
  e = calloc(1, sizeof(*e));
  if (e == NULL) return ga_err_sys(ctx->err, "calloc");
  e->fname = fname;
  e->key = key;
  e->fn = got;
  e->next = (lm_entry *)ctx->lm_cache;
  ctx->lm_cache = e;
  *fn = &e->fn;
  return GA_NO_ERROR;
}

void ga_lm_cache_free(gpucontext *ctx) {
  lm_entry *e = (lm_entry *)ctx->lm_cache, *n;
  ctx->lm_cache = NULL;
  for (; e != NULL; e = n) {
    n = e->next;
    free(e);
  }
}

/* --------------------------------------------------------------- workspaces */

int ga_lm_capturing(gpucontext *ctx) {
  CUstreamCaptureStatus st = CU_STREAM_CAPTURE_STATUS_NONE;
  ga_ctx_enter(ctx);
  ga_cu.p_cuStreamIsCapturing(ctx->s, &st);
  ga_ctx_exit(ctx);
  return st != CU_STREAM_CAPTURE_STATUS_NONE;
}

int ga_workspace_need(gpucontext *ctx, ga_workspace *ws, size_t bytes) {
  gpudata *b;
  int err = GA_NO_ERROR;
  if (bytes <= ws->sz) return GA_NO_ERROR;
  if (ga_lm_capturing(ctx))
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR,
                      "The operator's workspace cannot grow while a graph is captured: call it "
                      "once with these sizes before");
  if (bytes < 2 * ws->sz) bytes = 2 * ws->sz; /* all that was kept adds up to less than what is in use */
  if (ws->cur != NULL) {
    gpudata **old = realloc(ws->old, (ws->nold + 1) * sizeof(*old));
    if (old == NULL) return ga_err_sys(ctx->err, "realloc");
    ws->old = old;
  }
  b = gpudata_alloc(ctx, bytes, NULL, 0, &err);
  if (b == NULL) return err;
  if (ws->cur != NULL) ws->old[ws->nold++] = ws->cur;
  ws->cur = b;
  ws->sz = bytes;
  return GA_NO_ERROR;
}

void ga_workspace_free(ga_workspace *ws) {
  unsigned int i;
  for (i = 0; i < ws->nold; i++) gpudata_release(ws->old[i]);
  free(ws->old);
  if (ws->cur != NULL) gpudata_release(ws->cur);
  memset(ws, 0, sizeof(*ws));
}

/* --------------------------------------------------------------- error word */

CUdeviceptr ga_lm_err_word(gpucontext *ctx) { return ctx->errbuf->ptr + sizeof(int); }

int ga_lm_err_take(gpucontext *ctx, const char *what) {
  int set = 0, err;
  err = gpudata_read(&set, ctx->errbuf, sizeof(int), sizeof(int));
  if (err != GA_NO_ERROR || set == 0) return err;
  set = 0;
  err = gpudata_write(ctx->errbuf, sizeof(int), &set, sizeof(int));
  if (err != GA_NO_ERROR) return err;
  return ga_err_set(ctx->err, GA_VALUE_ERROR, what);
}

/* ----------------------------------------------------------------- geometry */

void ga_lm_geometry(unsigned long long nv, unsigned most, unsigned block[3], unsigned int *ny) {
  unsigned long long y = (nv + most - 1) / most, x;
  if (nv == 0) y = 1;
  x = (nv + y - 1) / y;
  if (x > 16) x = (x + 31) / 32 * 32;
  else {
    unsigned long long p = 1;
    while (p < x) p *= 2;
    x = p;
  }
  block[0] = (unsigned)x;
  block[1] = (unsigned)(256 / x);
  block[2] = 1;
  *ny = (unsigned)((nv + x - 1) / x);
  if (*ny == 0) *ny = 1;
}
