#define MC_T double
#include "rms_norm_inst.cuh"
