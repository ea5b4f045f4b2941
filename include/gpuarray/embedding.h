/* Token embedding: rows of a table by id, and the gradient of the table.
 *
 * The reference has the plain gather only (GpuArray_take1, src/gpuarray/array.h:355);
 * these add the scale, the padding id, strided ids of any rank and the adjoint.
 *
 *   out[t, :]     = scale * table[row(ids[t]), :]
 *   dtable[v, :]  = scale * sum over {t : row(ids[t]) = v} of dout[t, :]
 *
 * with t running over all dimensions of `ids`. row(i) is i, or i + V for a
 * negative i, V the rows of the table: the rule of GpuArray_take1.
 *
 *  - Element types are GA_HALF, GA_FLOAT and GA_DOUBLE in any mixture; ids are
 *    GA_INT, GA_UINT, GA_LONG or GA_ULONG. Products and sums are taken in float,
 *    or in double where an array is GA_DOUBLE, and rounded once when written.
 *    scale is finite as a float.
 *  - Offsets and strides of all arrays are honoured (adjacent row elements on
 *    16- or 32-byte boundaries are fastest). Dimensions of ids that lie one
 *    behind the other in both arrays count as one; more than four that do not
 *    are GA_UNSUPPORTED_ERROR. A destination must not overlap the other
 *    arrays, nor may two of its elements share a place.
 *  - GA_EMBED_PAD: tokens whose id equals `pad` (compared before the rule for
 *    negative ids; a GA_ULONG id of 2^63 and more by its bits) give a row of
 *    zeros and add nothing to the gradient.
 *  - An id outside the table leaves its row of `out` as it was and adds nothing
 *    to the gradient. With GA_EMBED_CHECK the call waits for the result and
 *    returns GA_VALUE_ERROR for it; without, it is not reported and nothing
 *    waits. A checked call cannot be captured into a CUDA graph
 *    (GA_UNSUPPORTED_ERROR). */
#ifndef GPUARRAY_EMBEDDING_H
#define GPUARRAY_EMBEDDING_H

#include <gpuarray/array.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GA_EMBED_PAD        0x0001
#define GA_EMBED_CHECK      0x0002
#define GA_EMBED_ACCUMULATE 0x0004 /* gradient only */

/* out: the dimensions of ids followed by one of table's row length; table: 2-d.
 * Enqueues on the context's stream and returns (unless GA_EMBED_CHECK). */
GPUARRAY_PUBLIC int GpuArray_embed(GpuArray *out, const GpuArray *table, const GpuArray *ids,
                                   double scale, ssize_t pad, int flags);

/* The gradient operator; it owns the workspace in which the tokens are sorted.
 * Calls of one operator must not overlap on the device (replays of graphs that
 * captured it included): use one operator for each. Its workspace only grows,
 * and memory that a captured graph may refer to is kept until
 * GpuEmbedGrad_free. */
typedef struct _GpuEmbedGrad GpuEmbedGrad;

GPUARRAY_PUBLIC int GpuEmbedGrad_new(GpuEmbedGrad **eg, gpucontext *ctx);
GPUARRAY_PUBLIC void GpuEmbedGrad_free(GpuEmbedGrad *eg);

/* dtable: 2-d, every row is written (rows that no token names with zeros);
 * with GA_EMBED_ACCUMULATE the sums are added to what is there and only the
 * rows that tokens name are touched. dout: the dimensions of ids followed by
 * one of dtable's row length. Tokens are summed in an order that the ids alone
 * decide, so equal calls give equal bits. At most 2^31 - 1 tokens and rows
 * (GA_XLARGE_ERROR). */
GPUARRAY_PUBLIC int GpuEmbedGrad_call(GpuEmbedGrad *eg, GpuArray *dtable, const GpuArray *dout,
                                      const GpuArray *ids, double scale, ssize_t pad, int flags);

#ifdef __cplusplus
}
#endif
#endif
