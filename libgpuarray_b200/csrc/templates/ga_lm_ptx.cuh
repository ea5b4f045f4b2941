/* Instructions the language-model kernels use beyond the shared vocabulary of
 * cluda.h. */
#ifndef GA_LM_PTX_CUH
#define GA_LM_PTX_CUH
#include "cluda.h"

/* 2^x, flushing results below the smallest normal number to zero */
static __device__ __forceinline__ float ga__ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
/* max(a, b) that is NaN when either is (fmaxf drops NaNs) */
static __device__ __forceinline__ float ga__max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
/* larger of two pairs of halves, NaNs dropped where the other is a number */
static __device__ __forceinline__ unsigned int ga__max_h2(unsigned int a, unsigned int b) {
  unsigned int r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
static __device__ __forceinline__ void ga__unpack_h2(unsigned int w, float &lo, float &hi) {
  asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;}"
      : "=f"(lo), "=f"(hi)
      : "r"(w));
}
static __device__ __forceinline__ unsigned int ga__pack_h2(float lo, float hi) {
  unsigned int w;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}
/* a double as half, with one rounding */
static __device__ __forceinline__ unsigned short ga__half_bits(double x) {
  unsigned short w;
  asm("cvt.rn.f16.f64 %0, %1;" : "=h"(w) : "d"(x));
  return w;
}

/* Two floats handled by one instruction (sm_100: packed add, multiply, fused multiply-add) */
struct ga__f2 {
  unsigned long long w;
};
static __device__ __forceinline__ ga__f2 ga__f2_of(float a, float b) {
  ga__f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.w) : "f"(a), "f"(b));
  return r;
}
static __device__ __forceinline__ void ga__f2_to(ga__f2 v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v.w));
}
static __device__ __forceinline__ ga__f2 ga__f2_add(ga__f2 a, ga__f2 b) {
  ga__f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}
static __device__ __forceinline__ ga__f2 ga__f2_mul(ga__f2 a, ga__f2 b) {
  ga__f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}
static __device__ __forceinline__ ga__f2 ga__f2_fma(ga__f2 a, ga__f2 b, ga__f2 c) {
  ga__f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.w) : "l"(a.w), "l"(b.w), "l"(c.w));
  return r;
}

/* 32 bytes of global memory by one access (p 32-byte aligned; sm_100) */
static __device__ __forceinline__ void ga__ld32(unsigned int w[8], const char *p) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
static __device__ __forceinline__ void ga__st32(char *p, const unsigned int w[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

/* The two halves of ga__grid_dependency_sync(), for a kernel that does not depend on its
 * predecessor in the stream but on what came before that one. */
static __device__ __forceinline__ void ga__grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
static __device__ __forceinline__ void ga__grid_dependency_release() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

/* Sum over the warp, the same in every lane */
static __device__ __forceinline__ unsigned int ga__warp_sum_u32(unsigned int v) {
  return __reduce_add_sync(0xffffffffu, v);
}

/* Shared memory of a kernel: one struct, of fixed size or with a tail whose size the launch gives */
#define GA_LM_SHARED(type, name) __shared__ type name
#define GA_LM_SHARED_DYNAMIC(type, name)                          \
  extern __shared__ unsigned long long ga__dynamic_shared[];      \
  type &name = *reinterpret_cast<type *>(ga__dynamic_shared)

/* ---- thread-block clusters ---- */
static __device__ __forceinline__ unsigned int ga__cluster_rank() {
  unsigned int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
/* Barrier over the cluster's threads in two halves; what each wrote to any CTA's shared
 * memory before its arrival is visible to all after their wait. */
static __device__ __forceinline__ void ga__cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
static __device__ __forceinline__ void ga__cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
/* Stores 8 bytes at the place that `p` (this CTA's shared memory) has in CTA `rank`'s. */
static __device__ __forceinline__ void ga__cluster_put(unsigned long long *p, unsigned int rank,
                                                       unsigned long long v) {
  const unsigned int s = (unsigned int)__cvta_generic_to_shared(p);
  asm volatile("{.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\t"
               "st.shared::cluster.u64 [a], %2;}" ::"r"(s), "r"(rank), "l"(v)
               : "memory");
}
/* The same with 4 bytes. */
static __device__ __forceinline__ void ga__cluster_put(unsigned int *p, unsigned int rank,
                                                       unsigned int v) {
  const unsigned int s = (unsigned int)__cvta_generic_to_shared(p);
  asm volatile("{.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\t"
               "st.shared::cluster.u32 [a], %2;}" ::"r"(s), "r"(rank), "r"(v)
               : "memory");
}
#endif
