#define MC_T __half
#include "rms_norm_inst.cuh"
