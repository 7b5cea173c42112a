#define MC_T float
#define MC_G float
#include "rms_norm_inst.cuh"
