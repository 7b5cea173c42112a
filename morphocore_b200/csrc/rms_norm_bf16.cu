#define MC_T __nv_bfloat16
#define MC_G __nv_bfloat16
#include "rms_norm_inst.cuh"
