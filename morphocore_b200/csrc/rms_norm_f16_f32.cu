#define MC_T __half
#define MC_G float
#include "rms_norm_inst.cuh"
