// Norms over rows: f32 x, f16 y.
#include "layer_norm_kernels.h"

TERRA_NORM_DEFINE(f32, F32, f16, F16)
