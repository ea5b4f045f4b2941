/* Build-time instantiation: log probabilities and entropy of half rows, one CTA each. */
#define GA_LP_BUILD_ROWS
#define GA_LP_Z_T ga_half
#define GA_LP_ZTYPE 0
#define GA_LP_I_T ga_int
#define GA_LP_ND 1
#define GA_LP_CONTIG 1
#define GA_LP_ENT 1
#define GA_LP_THREADS 128
#define GA_LP_GROUP 128
#define GA_LP_CLUSTER 1
#define GA_LP_TOP 0
#define GA_LP_FOLD 1
#include "ga_logprobs.cuh"
