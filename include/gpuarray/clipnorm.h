/* The norm over a list of arrays (a step's gradients) and the arrays scaled so
 * that it does not exceed a limit, in two launches however many arrays there
 * are. No counterpart in the reference, where this is a reduction and an
 * elementwise call for each array.
 *
 *   norm   = |scale| * sqrt(sum over all arrays and elements of src^2)
 *   dst[i] = src[i] * scale * min(1, limit / norm)
 *
 *  - Arrays are GA_HALF, GA_FLOAT or GA_DOUBLE, each its own; dst[i] has the type
 *    of src[i], or GA_FLOAT where src[i] is GA_HALF. They are one segment in
 *    memory (C or Fortran order, dst[i] the same as src[i]) of any alignment
 *    that their type has; anything else is GA_INVALID_ERROR. Arrays without
 *    elements are allowed. Fastest where dst[i] starts as many elements past a
 *    16-byte boundary as src[i] (16 or 32 bytes for halfs into floats): else
 *    each element is stored by itself, floats in 1.06 and halfs in 3.3 times
 *    the time of 10^8 of them.
 *  - Squares are summed in double in an order that the sizes alone decide:
 *    equal calls give equal bits, and no finite float overflows (doubles beyond
 *    1e154 do: an infinite norm). Products with the factor are rounded to the
 *    type of dst whatever the factor's size.
 *  - A NaN anywhere gives a NaN norm and NaN in every dst; an infinity gives
 *    an infinite norm, zeros for finite elements and NaN for infinite ones
 *    (limit infinite: nothing is clipped).
 *  - dst[i] may be src[i] (nothing is written where the factor is 1); no other
 *    two arrays may overlap where one of them is a destination, the norm among
 *    them (GA_VALUE_ERROR). */
#ifndef GPUARRAY_CLIPNORM_H
#define GPUARRAY_CLIPNORM_H

#include <gpuarray/array.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GA_CLIPNORM_MAX_ARRAYS 32768

/* The operator owns the workspace of the sum. Calls of one operator must not
 * overlap on the device (replays of graphs that captured it included): use one
 * operator for each. */
typedef struct _GpuClipNorm GpuClipNorm;

GPUARRAY_PUBLIC int GpuClipNorm_new(GpuClipNorm **cn, gpucontext *ctx);
GPUARRAY_PUBLIC void GpuClipNorm_free(GpuClipNorm *cn);

/* norm: 0-d, GA_FLOAT or GA_DOUBLE. dst: n destinations, or NULL for the norm
 * alone. src: n arrays. scale is finite, limit 0 or more (infinity: no limit).
 * n may be 0. Enqueues on the context's stream and returns. */
GPUARRAY_PUBLIC int GpuClipNorm_call(GpuClipNorm *cn, GpuArray *norm, GpuArray *const *dst,
                                     const GpuArray *const *src, unsigned int n, double scale,
                                     double limit);

#ifdef __cplusplus
}
#endif
#endif
