/* Build-time instantiation: gradient of a half table, tokens sorted by a cluster. */
#define GA_EM_BUILD_GRAD
#define GA_EM_A_T ga_half
#define GA_EM_O_T ga_half
#define GA_EM_I_T ga_long
#define GA_EM_F_T ga_float
#define GA_EM_E 8
#define GA_EM_C 1
#define GA_EM_ND 2
#define GA_EM_ACCUMULATE 0
#define GA_EG_ROUNDS 2
#define GA_EG_CLUSTER 8
#include "ga_embed.cuh"
