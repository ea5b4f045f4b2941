/* Log probabilities, entropy, alternatives and their gradient
 * (include/gpuarray/logprobs.h; kernels in templates/ga_logprobs.cuh). */
#include <math.h>
#include "private.h"

typedef struct lp_layout { /* the templates' ga__lp_layout */
  unsigned long long rows;
  unsigned int v, top;
  float scale;
  int has_ignore;
  long long ignore;
  unsigned long long dims[GA_LM_MAXD];
  long long z_str[GA_LM_MAXD], t_str[GA_LM_MAXD];
  long long z_col;
  long long o_str[5][GA_LM_MAXD];
  long long o_col[5];
} lp_layout;

struct _GpuLogProbs {
  gpucontext *ctx;
  int z_tc, i_tc;
  unsigned int top;
};

typedef struct lp_variant {
  int z_tc, i_tc, g_tc, grad, contig, ent, top, fold;
  unsigned threads, group, cluster, nd;
} lp_variant;

#define LP_LOG2E 1.4426950408889634f /* GA_LP_LOG2E of the template */
#define LP_U 4 /* vectors of a thread in one step: GA_LP_U of the template */

static uint64_t variant_key(const lp_variant *v) {
  return (uint64_t)v->z_tc | (uint64_t)v->i_tc << 8 | (uint64_t)v->g_tc << 16 |
         (uint64_t)(v->threads / 32) << 24 | (uint64_t)(v->group / 32) << 32 |
         (uint64_t)v->cluster << 40 | (uint64_t)v->nd << 48 | (uint64_t)v->grad << 56 |
         (uint64_t)v->contig << 57 | (uint64_t)v->ent << 58 | (uint64_t)v->top << 59 | (uint64_t)v->fold << 60;
}

static void emit(ga_strb *sb, uint64_t key) {
  const int z = (int)(key & 0xff), i = (int)((key >> 8) & 0xff), g = (int)((key >> 16) & 0xff);
  const int grad = (int)((key >> 56) & 1);
  ga_strb_printf(sb,
                 "#include \"cluda.h\"\n#define %s\n#define GA_LP_Z_T %s\n#define GA_LP_ZTYPE %d\n"
                 "#define GA_LP_I_T %s\n#define GA_LP_ND %u\n#define GA_LP_CONTIG %u\n"
                 "#define GA_LP_ENT %u\n",
                 grad ? "GA_LP_BUILD_GRAD" : "GA_LP_BUILD_ROWS", ga_ctype(z), z == GA_FLOAT,
                 ga_ctype(i), (unsigned)((key >> 48) & 0xff), (unsigned)((key >> 57) & 1),
                 (unsigned)((key >> 58) & 1));
  if (grad)
    ga_strb_printf(sb, "#define GA_LP_G_T %s\n#define GA_LP_GTYPE %d\n", ga_ctype(g), g == GA_FLOAT);
  else
    ga_strb_printf(sb,
                   "#define GA_LP_THREADS %u\n#define GA_LP_GROUP %u\n#define GA_LP_CLUSTER %u\n"
                   "#define GA_LP_TOP %u\n#define GA_LP_FOLD %u\n",
                   (unsigned)((key >> 24) & 0xff) * 32, (unsigned)((key >> 32) & 0xff) * 32,
                   (unsigned)((key >> 40) & 0xff), (unsigned)((key >> 59) & 1), (unsigned)((key >> 60) & 1));
  ga_strb_puts(sb, "#include \"ga_logprobs.cuh\"\n");
}

int GpuLogProbs_new(GpuLogProbs **lp, gpucontext *ctx, int typecode, int id_typecode,
                    unsigned int top) {
  GpuLogProbs *r;
  if (lp == NULL) return GA_INVALID_ERROR;
  *lp = NULL;
  if (ctx == NULL) return ga_err_set(ga_global_err, GA_INVALID_ERROR, "GpuLogProbs_new: no context");
  if (typecode != GA_HALF && typecode != GA_FLOAT)
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR, "Logits must be half or float");
  if (!ga_lm_is_id(id_typecode))
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR, "Token ids must be 32- or 64-bit integers");
  if (top > GA_LOGPROBS_MAX_TOP)
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "At most %d alternatives", GA_LOGPROBS_MAX_TOP);
  r = calloc(1, sizeof(*r));
  if (r == NULL) return ga_err_sys(ctx->err, "calloc");
  r->ctx = ctx;
  r->z_tc = typecode;
  r->i_tc = id_typecode;
  r->top = top;
  ctx->refcnt++;
  *lp = r;
  return GA_NO_ERROR;
}

void GpuLogProbs_free(GpuLogProbs *lp) {
  gpucontext *ctx;
  if (lp == NULL) return;
  ctx = lp->ctx;
  free(lp);
  ga_ctx_unref(ctx);
}

/* An array with the rows' dimensions (and one of `last`, unless that is 0); the checks of
 * ga_lm_check and the type. */
static int check_array(gpucontext *ctx, const GpuArray *a, const char *what, int dest, int tc,
                       const GpuArray *logits, size_t last) {
  const unsigned nd = logits->nd - 1;
  int err = ga_lm_check(ctx, a, what, dest);
  if (err != GA_NO_ERROR) return err;
  if (a->typecode != tc)
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "%s has type %d, expected %d", what, a->typecode, tc);
  if (a->nd != nd + (last != 0) || !ga_lm_same_dims(a, logits, nd) ||
      (last != 0 && a->dimensions[nd] != last))
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "%s has not the shape that the logits give it", what);
  return GA_NO_ERROR;
}

static int check_common(GpuLogProbs *lp, const GpuArray *logits, double scale, int flags) {
  gpucontext *ctx = lp->ctx;
  int err = ga_lm_check(ctx, logits, "logits", 0);
  if (err != GA_NO_ERROR) return err;
  if (logits->typecode != lp->z_tc)
    return ga_err_fmt(ctx->err, GA_VALUE_ERROR, "logits has type %d, the operator takes %d",
                      logits->typecode, lp->z_tc);
  if (logits->nd == 0 || logits->dimensions[logits->nd - 1] == 0)
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "logits has no vocabulary axis");
  if (logits->dimensions[logits->nd - 1] >= (1UL << 28))
    return ga_err_set(ctx->err, GA_XLARGE_ERROR, "The vocabulary has 2^28 entries or more");
  if (!(scale > 0) || isinf((float)scale * LP_LOG2E) || (float)scale == 0) /* the kernels' exponents */
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "scale must be positive, and finite as a float times log2 e");
  if (flags & ~(GA_LOGPROBS_IGNORE | GA_LOGPROBS_CHECK))
    return ga_err_fmt(ctx->err, GA_INVALID_ERROR, "Unknown flags 0x%x", flags);
  if (ISSET(flags, GA_LOGPROBS_CHECK) && ga_lm_capturing(ctx))
    return ga_err_set(ctx->err, GA_UNSUPPORTED_ERROR,
                      "A checked call waits and cannot be captured into a graph");
  return GA_NO_ERROR;
}

/* The layout for logits, targets and five more arrays (any of them but the first may be NULL);
 * last: they have an axis beyond the rows'. */
static int fill(GpuLogProbs *lp, lp_layout *L, unsigned *nd, const GpuArray *logits,
                const GpuArray *targets, GpuArray *const arr[5], const int last[5], double scale,
                ssize_t ignore, int flags) {
  const ssize_t *str[7];
  long long out[7][GA_LM_MAXD];
  ga_lead lead;
  unsigned k;
  int err;
  memset(L, 0, sizeof(*L));
  str[0] = logits->strides;
  str[1] = targets != NULL ? targets->strides : NULL;
  for (k = 0; k < 5; k++) str[2 + k] = arr[k] != NULL ? arr[k]->strides : NULL;
  err = ga_lm_lead(lp->ctx, logits->nd - 1, logits->dimensions, 7, str, &lead, out);
  if (err != GA_NO_ERROR) return err;
  *nd = lead.nd;
  L->rows = lead.count;
  L->v = (unsigned)logits->dimensions[logits->nd - 1];
  L->top = lp->top;
  L->scale = (float)scale;
  L->has_ignore = ISSET(flags, GA_LOGPROBS_IGNORE);
  L->ignore = ignore;
  memcpy(L->dims, lead.dims, sizeof(L->dims));
  memcpy(L->z_str, out[0], sizeof(L->z_str));
  memcpy(L->t_str, out[1], sizeof(L->t_str));
  L->z_col = logits->strides[logits->nd - 1];
  for (k = 0; k < 5; k++) {
    memcpy(L->o_str[k], out[2 + k], sizeof(L->o_str[k]));
    if (arr[k] != NULL && last[k]) L->o_col[k] = arr[k]->strides[arr[k]->nd - 1];
  }
  if (L->rows > 0x3fffffffULL) /* times CTAs of a cluster, in a grid of 2^31 - 1 */
    return ga_err_set(lp->ctx->err, GA_XLARGE_ERROR, "More than 2^30 - 1 rows in one call");
  return GA_NO_ERROR;
}

static CUdeviceptr at(const GpuArray *a) { return a == NULL ? 0 : a->data->ptr + a->offset; }

/* most vectors a row can touch: its first one may start anywhere in a 16-byte word */
static unsigned long long row_vectors(const lp_layout *L, unsigned e) {
  return e == 1 ? L->v : ((unsigned long long)L->v + 2 * (e - 1)) / e;
}

/* Threads and CTAs for a row of nv vectors. Many short rows: a warp each, which has nothing to wait
 * for but itself ((16384, 4000) halfs 33 us, with 5 alternatives 49; a CTA each 47 and 88). Many
 * long rows: CTAs of 128 threads, 8 of them an SM, as more threads only make the last wave longer
 * ((2047, 50021) halfs: 39 us with 128, 41 with 256). Fewer: 256 or 512, where the row gives each
 * thread enough to do ((700, 131072) halfs: 35 us with 512, 39 with 256, 51 with 128), and 512
 * where all rows are on the device at once; then up to 8 CTAs in a cluster, as long as the device
 * holds them and each has a full step of loads (3 rows of 131072 halfs, 20 alternatives: 8.6 us;
 * one CTA for a row 13.2). */
static void choose_shape(lp_variant *v, unsigned long long rows, unsigned long long nv, unsigned num_sms) {
  const unsigned long long device = (unsigned long long)num_sms * 1024; /* threads it holds at once */
  v->threads = v->top ? 128 : 256; /* a warp's lists are 7 KiB of shared memory */
  v->group = 32;
  v->cluster = 1;
  if (nv <= 64 || (nv <= (v->top ? 1024u : 2048u) && rows >= (unsigned long long)num_sms * 16)) return;
  v->threads = 128;
  if (rows <= (unsigned long long)num_sms * 8 && nv >= 256 * LP_U * 3) v->threads = 256;
  if (rows <= (unsigned long long)num_sms * 8 && nv >= 512 * LP_U * 6) v->threads = 512;
  if (rows * 512 <= device && nv >= 512 * LP_U) v->threads = 512;
  while (v->cluster < 8 && rows * v->cluster * 2 * v->threads <= device &&
         nv >= (unsigned long long)v->cluster * 2 * v->threads * LP_U)
    v->cluster *= 2;
  v->group = v->threads;
}

#define LP_FOLD_SCALE 64.0f /* halfs times this and log2 e stay below 2^23 */

int GpuLogProbs_call(GpuLogProbs *lp, GpuArray *logp, GpuArray *entropy, GpuArray *stats,
                     GpuArray *top_logp, GpuArray *top_ids, const GpuArray *logits,
                     const GpuArray *targets, double scale, ssize_t ignore, int flags) {
  gpucontext *ctx;
  GpuArray *arr[5];
  static const int last[5] = {0, 0, 1, 1, 1};
  lp_layout L;
  lp_variant v;
  const ga_function *fn;
  CUdeviceptr p[8];
  void *params[10];
  unsigned grid[3] = {1, 1, 1}, block[3] = {256, 1, 1}, i, e;
  size_t es;
  int err;

  if (lp == NULL) return GA_INVALID_ERROR;
  ctx = lp->ctx;
  if ((err = check_common(lp, logits, scale, flags)) != GA_NO_ERROR) return err;
  if (logp == NULL && entropy == NULL && stats == NULL && top_logp == NULL && top_ids == NULL)
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "No destination");
  if ((logp != NULL) != (targets != NULL))
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "logp and targets go together");
  if ((top_logp != NULL || top_ids != NULL) && lp->top == 0)
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "The operator was made without alternatives");
  if (lp->top > logits->dimensions[logits->nd - 1] && (top_logp != NULL || top_ids != NULL))
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "More alternatives than vocabulary entries");
  if ((logp != NULL && ((err = check_array(ctx, logp, "logp", 1, GA_FLOAT, logits, 0)) != GA_NO_ERROR ||
                        (err = check_array(ctx, targets, "targets", 0, lp->i_tc, logits, 0)) != GA_NO_ERROR)) ||
      (entropy != NULL && (err = check_array(ctx, entropy, "entropy", 1, GA_FLOAT, logits, 0)) != GA_NO_ERROR) ||
      (stats != NULL && (err = check_array(ctx, stats, "stats", 1, GA_FLOAT, logits, 2)) != GA_NO_ERROR) ||
      (top_logp != NULL &&
       (err = check_array(ctx, top_logp, "top_logp", 1, GA_FLOAT, logits, lp->top)) != GA_NO_ERROR) ||
      (top_ids != NULL &&
       (err = check_array(ctx, top_ids, "top_ids", 1, lp->i_tc, logits, lp->top)) != GA_NO_ERROR))
    return err;
  arr[0] = logp;
  arr[1] = entropy;
  arr[2] = stats;
  arr[3] = top_logp;
  arr[4] = top_ids;
  memset(&v, 0, sizeof(v));
  err = fill(lp, &L, &v.nd, logits, targets, arr, last, scale, ignore, flags);
  if (err != GA_NO_ERROR || L.rows == 0) return err;

  es = gpuarray_get_elsize(lp->z_tc);
  v.z_tc = lp->z_tc;
  v.i_tc = lp->i_tc;
  v.contig = L.z_col == (long long)es || L.v == 1;
  if (L.v == 1) L.z_col = (long long)es;
  v.ent = entropy != NULL;
  v.top = top_logp != NULL || top_ids != NULL;
  v.fold = lp->z_tc == GA_HALF && L.scale <= LP_FOLD_SCALE;
  e = v.contig ? 16 / (unsigned)es : 1;
  choose_shape(&v, L.rows, row_vectors(&L, e), ctx->num_sms);
  err = ga_lm_kernel(ctx, "ga_lp_rows", variant_key(&v), emit, &fn);
  if (err != GA_NO_ERROR) return err;
  block[0] = v.threads;
  grid[0] = (unsigned)((L.rows + v.threads / v.group - 1) / (v.threads / v.group)) * v.cluster;
  p[0] = at(logits);
  p[1] = at(targets);
  for (i = 0; i < 5; i++) p[2 + i] = at(arr[i]);
  p[7] = ISSET(flags, GA_LOGPROBS_CHECK) ? ga_lm_err_word(ctx) : 0;
  params[0] = &L;
  for (i = 0; i < 8; i++) params[1 + i] = &p[i];
  err = ga_launch(ctx, fn, grid, block, 0, params);
  if (err == GA_NO_ERROR && ISSET(flags, GA_LOGPROBS_CHECK))
    err = ga_lm_err_take(ctx, "A target is outside the vocabulary");
  return err;
}

#define LP_CTAS 16 /* of 256 threads, 3 of which an SM holds at once where logits are adjacent (80 registers
                      a thread; one word of it spilled for halfs without entropy and one leading dimension) */

int GpuLogProbs_grad(GpuLogProbs *lp, GpuArray *dlogits, const GpuArray *logits,
                     const GpuArray *targets, const GpuArray *stats, const GpuArray *dlogp,
                     const GpuArray *entropy, const GpuArray *dentropy, double scale,
                     ssize_t ignore, int flags) {
  gpucontext *ctx;
  GpuArray *arr[5];
  static const int last[5] = {1, 0, 0, 0, 1};
  lp_layout L;
  lp_variant v;
  const ga_function *fn;
  CUdeviceptr p[8];
  void *params[10];
  unsigned grid[3] = {1, 1, 1}, block[3], i, e;
  size_t es;
  int err;

  if (lp == NULL) return GA_INVALID_ERROR;
  ctx = lp->ctx;
  if ((err = check_common(lp, logits, scale, flags)) != GA_NO_ERROR ||
      (err = ga_lm_check(ctx, dlogits, "dlogits", 1)) != GA_NO_ERROR)
    return err;
  if (dlogits->typecode != lp->z_tc && dlogits->typecode != GA_FLOAT)
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "dlogits must be float or of the logits' type");
  if (dentropy != NULL && entropy == NULL)
    return ga_err_set(ctx->err, GA_VALUE_ERROR, "dentropy needs entropy");
  if ((err = check_array(ctx, dlogits, "dlogits", 1, dlogits->typecode, logits,
                         logits->dimensions[logits->nd - 1])) != GA_NO_ERROR ||
      (err = check_array(ctx, targets, "targets", 0, lp->i_tc, logits, 0)) != GA_NO_ERROR ||
      (err = check_array(ctx, stats, "stats", 0, GA_FLOAT, logits, 2)) != GA_NO_ERROR ||
      (err = check_array(ctx, dlogp, "dlogp", 0, GA_FLOAT, logits, 0)) != GA_NO_ERROR ||
      (dentropy != NULL &&
       ((err = check_array(ctx, entropy, "entropy", 0, GA_FLOAT, logits, 0)) != GA_NO_ERROR ||
        (err = check_array(ctx, dentropy, "dentropy", 0, GA_FLOAT, logits, 0)) != GA_NO_ERROR)))
    return err;
  arr[0] = (GpuArray *)stats;
  arr[1] = (GpuArray *)dlogp;
  arr[2] = dentropy != NULL ? (GpuArray *)entropy : NULL;
  arr[3] = (GpuArray *)dentropy;
  arr[4] = dlogits;
  memset(&v, 0, sizeof(v));
  err = fill(lp, &L, &v.nd, logits, targets, arr, last, scale, ignore, flags);
  if (err != GA_NO_ERROR || L.rows == 0) return err;

  es = gpuarray_get_elsize(lp->z_tc);
  v.z_tc = lp->z_tc;
  v.i_tc = lp->i_tc;
  v.g_tc = dlogits->typecode;
  v.grad = 1;
  v.contig = L.z_col == (long long)es || L.v == 1;
  if (L.v == 1) L.z_col = (long long)es;
  v.ent = dentropy != NULL;
  e = v.contig ? 16 / (unsigned)es : 1;
  err = ga_lm_kernel(ctx, "ga_lp_grad", variant_key(&v), emit, &fn);
  if (err != GA_NO_ERROR) return err;
  ga_lm_geometry((row_vectors(&L, e) + LP_U - 1) / LP_U, 256, block, &grid[1]);
  grid[0] = (unsigned)((L.rows + block[1] - 1) / block[1]);
  /* A CTA takes as many steps along its row as leave LP_CTAS for every SM. */
  {
    unsigned long long want = ((unsigned long long)ctx->num_sms * LP_CTAS + grid[0] - 1) / grid[0];
    if (grid[1] > want) grid[1] = (unsigned)want;
  }
  p[0] = at(dlogits);
  p[1] = at(logits);
  p[2] = at(targets);
  for (i = 0; i < 4; i++) p[3 + i] = at(arr[i]);
  p[7] = ISSET(flags, GA_LOGPROBS_CHECK) ? ga_lm_err_word(ctx) : 0;
  params[0] = &L;
  for (i = 0; i < 8; i++) params[1 + i] = &p[i];
  err = ga_launch(ctx, fn, grid, block, 0, params);
  if (err == GA_NO_ERROR && ISSET(flags, GA_LOGPROBS_CHECK))
    err = ga_lm_err_take(ctx, "A target is outside the vocabulary");
  return err;
}
