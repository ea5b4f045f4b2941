/* Build-time instantiation: gradient of log probabilities and entropy for half logits. */
#define GA_LP_BUILD_GRAD
#define GA_LP_Z_T ga_half
#define GA_LP_ZTYPE 0
#define GA_LP_I_T ga_int
#define GA_LP_G_T ga_half
#define GA_LP_GTYPE 0
#define GA_LP_ND 1
#define GA_LP_CONTIG 1
#define GA_LP_ENT 1
#include "ga_logprobs.cuh"
