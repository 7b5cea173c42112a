#define MC_T __nv_bfloat16
#define MC_G float
#include "rms_norm_inst.cuh"
