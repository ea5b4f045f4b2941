/* Host stand-in for templates/ga_lm_ptx.cuh under the SIMT emulator: the same
 * operations in plain C++, and the intrinsics the language-model templates use
 * beyond those of simt_emul.h. The CTAs of a cluster run together
 * (simt_cluster.cpp), each with shared memory of its own. */
#ifndef GA_LM_PTX_CUH
#define GA_LM_PTX_CUH
#include "cluda.h"

static inline float __uint_as_float(unsigned int u) {
  float f;
  memcpy(&f, &u, 4);
  return f;
}
static inline unsigned int __float_as_uint(float f) {
  unsigned int u;
  memcpy(&u, &f, 4);
  return u;
}
template <typename T>
static inline T __shfl_xor_sync(unsigned, T v, int mask, int width = 32) {
  const unsigned lane = simt::cur->linear % 32;
  return simt__shfl(v, (lane % (unsigned)width) ^ (unsigned)mask, width);
}
template <typename T>
static inline T __shfl_up_sync(unsigned, T v, int delta, int width = 32) {
  const unsigned lane = simt::cur->linear % 32, in = lane % (unsigned)width;
  return simt__shfl(v, in >= (unsigned)delta ? in - (unsigned)delta : in, width);
}
static inline unsigned int __ballot_sync(unsigned, int pred) {
  const unsigned w = simt::cur->linear / 32, lane = simt::cur->linear % 32, n = simt::warp_lanes(w);
  simt::warp_slot[w][lane] = pred != 0;
  simt::warp_barrier(w, n);
  unsigned int r = 0;
  for (unsigned l = 0; l < n; l++) r |= (unsigned int)simt::warp_slot[w][l] << l;
  simt::warp_barrier(w, n);
  return r;
}
static inline float __fmul_rn(float a, float b) { return a * b; }
static inline int __popc(unsigned int v) { return __builtin_popcount(v); }
static inline int __ffs(unsigned int v) { return __builtin_ffs((int)v); }
static inline unsigned int ga__warp_sum_u32(unsigned int v) {
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

static inline float ga__ex2(float x) {
  const float r = exp2f(x);
  return r < 1.17549435e-38f ? 0.0f : r;
}
static inline float ga__max_nan(float a, float b) {
  if (a != a || b != b) return __uint_as_float(0x7fffffffu);
  return a > b ? a : b;
}
static inline void ga__unpack_h2(unsigned int w, float &lo, float &hi) {
  ga_half l, h;
  l.data = (ga_ushort)(w & 0xffffu);
  h.data = (ga_ushort)(w >> 16);
  lo = ga_half2float(l);
  hi = ga_half2float(h);
}
static inline unsigned int ga__pack_h2(float lo, float hi) {
  return (unsigned int)ga_float2half(lo).data | (unsigned int)ga_float2half(hi).data << 16;
}
static inline unsigned short ga__half_bits(double x) {
  const _Float16 v = (_Float16)x; /* one rounding to nearest even */
  unsigned short w;
  memcpy(&w, &v, 2);
  return w;
}
static inline unsigned int ga__max_h2(unsigned int a, unsigned int b) {
  float al, ah, bl, bh;
  ga__unpack_h2(a, al, ah);
  ga__unpack_h2(b, bl, bh);
  return ga__pack_h2(fmaxf(al, bl), fmaxf(ah, bh));
}
static inline void ga__ld32(unsigned int w[8], const char *p) {
  if ((size_t)p % 32 != 0) abort();
  memcpy(w, p, 32);
}
static inline void ga__st32(char *p, const unsigned int w[8]) {
  if ((size_t)p % 32 != 0) abort();
  memcpy(p, w, 32);
}
static inline void ga__grid_dependency_wait() {}
static inline void ga__grid_dependency_release() {}
struct ga__f2 {
  float a, b;
};
static inline ga__f2 ga__f2_of(float a, float b) { return ga__f2{a, b}; }
static inline void ga__f2_to(ga__f2 v, float &a, float &b) {
  a = v.a;
  b = v.b;
}
static inline ga__f2 ga__f2_add(ga__f2 x, ga__f2 y) { return ga__f2{x.a + y.a, x.b + y.b}; }
static inline ga__f2 ga__f2_mul(ga__f2 x, ga__f2 y) { return ga__f2{x.a * y.a, x.b * y.b}; }
static inline ga__f2 ga__f2_fma(ga__f2 x, ga__f2 y, ga__f2 z) {
  return ga__f2{fmaf(x.a, y.a, z.a), fmaf(x.b, y.b, z.b)};
}

/* ---- shared memory and clusters ---- */
namespace simt {
extern unsigned cluster_rank;   /* of the running CTA */
char *shared_of(unsigned rank); /* a CTA's shared memory */
void cluster_arrive();
void cluster_wait();
}
#define GA_LM_SHARED(type, name) type &name = *reinterpret_cast<type *>(simt::shared_of(simt::cluster_rank))
#define GA_LM_SHARED_DYNAMIC(type, name) GA_LM_SHARED(type, name)
#define __cluster_dims__(...)
static inline unsigned int ga__cluster_rank() { return simt::cluster_rank; }
static inline void ga__cluster_arrive() { simt::cluster_arrive(); }
static inline void ga__cluster_wait() { simt::cluster_wait(); }
template <typename T>
static inline void ga__cluster_put(T *p, unsigned int rank, T v) {
  const size_t at = (char *)p - simt::shared_of(simt::cluster_rank);
  if (at >= 256 * 1024) abort(); /* not in this CTA's shared memory */
  memcpy(simt::shared_of(rank) + at, &v, sizeof(T));
}
#endif
