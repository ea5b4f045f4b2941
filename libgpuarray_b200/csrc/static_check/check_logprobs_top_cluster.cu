/* Build-time instantiation: alternatives of float rows, eight CTAs for each. */
#define GA_LP_BUILD_ROWS
#define GA_LP_Z_T ga_float
#define GA_LP_ZTYPE 1
#define GA_LP_I_T ga_long
#define GA_LP_ND 1
#define GA_LP_CONTIG 1
#define GA_LP_ENT 0
#define GA_LP_THREADS 512
#define GA_LP_GROUP 512
#define GA_LP_CLUSTER 8
#define GA_LP_TOP 1
#define GA_LP_FOLD 0
#include "ga_logprobs.cuh"
