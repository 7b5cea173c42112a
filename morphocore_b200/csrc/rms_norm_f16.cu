#define MC_T __half
#define MC_G __half
#include "rms_norm_inst.cuh"
