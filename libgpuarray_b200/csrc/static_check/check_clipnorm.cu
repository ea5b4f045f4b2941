/* Build-time instantiation: norm and scaling over a list of up to 128 arrays. */
#define GA_CN_CAP 128
#include "ga_clipnorm.cuh"
