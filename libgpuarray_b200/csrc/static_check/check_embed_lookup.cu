/* Build-time instantiation: lookup of half rows by 32-bit ids, [batch, length] of a longer array. */
#define GA_EM_BUILD_LOOKUP
#define GA_EM_A_T ga_half
#define GA_EM_O_T ga_half
#define GA_EM_I_T ga_int
#define GA_EM_F_T ga_float
#define GA_EM_E 8
#define GA_EM_C 1
#define GA_EM_ND 2
#define GA_EM_ACCUMULATE 0
#include "ga_embed.cuh"
