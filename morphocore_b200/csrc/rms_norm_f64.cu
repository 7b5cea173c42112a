#define MC_T double
#define MC_G double
#include "rms_norm_inst.cuh"
