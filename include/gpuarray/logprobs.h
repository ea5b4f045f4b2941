/* Log probabilities of given tokens under rows of logits, with the entropy of
 * the rows and their most likely alternatives, in one pass over the logits;
 * and the gradient of the first two. No counterpart in the reference, where a
 * client writes this as several reductions and elementwise passes.
 *
 * For a row z of V logits, x = scale * z, p = softmax(x):
 *   logp    = ln p[target]
 *   entropy = -sum_j p_j ln p_j
 *   stats   = (max z, ln sum_j e^(x_j - scale max z)); their combination
 *             scale * stats[0] + stats[1] is the log-sum-exp of x
 *   top     = the `top` largest logits' ln p and indices, largest first, equal
 *             logits by the lower index, NaNs last
 *   dlogits_j = scale (dlogp (1[j = target] - p_j) - dentropy p_j (ln p_j + entropy))
 *
 *  - Logits are GA_HALF or GA_FLOAT; the last axis is the vocabulary (1 to
 *    2^28 - 1 entries), the others are the rows. Tokens are GA_INT, GA_UINT,
 *    GA_LONG or GA_ULONG. All other results and inputs are GA_FLOAT; dlogits is
 *    GA_FLOAT or the logits' type. Arithmetic is in float. scale is positive
 *    and at most 2.358e38, so that scale * log2 e is a float (GA_VALUE_ERROR).
 *    Differences of logits are taken before it: where two finite logits are
 *    further apart than the largest float, the lower one has probability 0.
 *  - Offsets and strides are honoured (rows' dimensions that lie one behind the
 *    other in all arrays count as one; more than four that do not are
 *    GA_UNSUPPORTED_ERROR); inputs of the gradient may have strides
 *    of 0 (one dlogp for all rows). Adjacent logits are fastest; rows may start
 *    at any element. dlogits may be the logits themselves; other overlaps of a
 *    destination are not allowed.
 *  - A row without a logit above -inf: logp and the alternatives' values are
 *    -inf, entropy 0, stats (-inf, -inf), gradient 0. A row that holds a NaN or
 *    +inf: NaN in all of them (the indices stay those of the largest numbers).
 *  - GA_LOGPROBS_IGNORE: rows whose target equals `ignore` (a GA_ULONG of 2^63
 *    and more by its bits) have logp 0, which has no gradient: the dlogp term is
 *    dropped whatever the row holds.
 *  - Any other target outside [0, V) gives a logp and a gradient row of NaN,
 *    whatever the row holds; with GA_LOGPROBS_CHECK the call also waits for the
 *    result and returns GA_VALUE_ERROR (not while a CUDA graph is captured:
 *    GA_UNSUPPORTED_ERROR). */
#ifndef GPUARRAY_LOGPROBS_H
#define GPUARRAY_LOGPROBS_H

#include <gpuarray/array.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GA_LOGPROBS_IGNORE 0x0001
#define GA_LOGPROBS_CHECK  0x0002
#define GA_LOGPROBS_MAX_TOP 32

typedef struct _GpuLogProbs GpuLogProbs;

/* typecode: of the logits; id_typecode: of targets and top_ids; top: number of
 * alternatives, 0 to GA_LOGPROBS_MAX_TOP. The operator holds no device memory:
 * its calls may overlap. */
GPUARRAY_PUBLIC int GpuLogProbs_new(GpuLogProbs **lp, gpucontext *ctx, int typecode,
                                    int id_typecode, unsigned int top);
GPUARRAY_PUBLIC void GpuLogProbs_free(GpuLogProbs *lp);

/* Any destination may be NULL, but not all. logp, entropy: the dimensions of
 * the rows; stats: those and one of 2; top_logp, top_ids: those and one of
 * `top`. targets: the dimensions of the rows; NULL without logp. */
GPUARRAY_PUBLIC int GpuLogProbs_call(GpuLogProbs *lp, GpuArray *logp, GpuArray *entropy,
                                     GpuArray *stats, GpuArray *top_logp, GpuArray *top_ids,
                                     const GpuArray *logits, const GpuArray *targets,
                                     double scale, ssize_t ignore, int flags);

/* stats and entropy are what GpuLogProbs_call wrote for the same logits and
 * scale; entropy is needed with dentropy only (both may be NULL). */
GPUARRAY_PUBLIC int GpuLogProbs_grad(GpuLogProbs *lp, GpuArray *dlogits, const GpuArray *logits,
                                     const GpuArray *targets, const GpuArray *stats,
                                     const GpuArray *dlogp, const GpuArray *entropy,
                                     const GpuArray *dentropy, double scale, ssize_t ignore,
                                     int flags);

#ifdef __cplusplus
}
#endif
#endif
