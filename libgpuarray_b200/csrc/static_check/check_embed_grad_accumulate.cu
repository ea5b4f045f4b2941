/* Build-time instantiation: float gradient of an odd width added to what is there. */
#define GA_EM_BUILD_GRAD
#define GA_EM_A_T ga_float
#define GA_EM_O_T ga_float
#define GA_EM_I_T ga_int
#define GA_EM_F_T ga_float
#define GA_EM_E 1
#define GA_EM_C 4
#define GA_EM_ND 1
#define GA_EM_ACCUMULATE 1
#define GA_EG_ROUNDS 1
#define GA_EG_CLUSTER 1
#include "ga_embed.cuh"
