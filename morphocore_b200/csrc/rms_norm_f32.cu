#define MC_T float
#include "rms_norm_inst.cuh"
