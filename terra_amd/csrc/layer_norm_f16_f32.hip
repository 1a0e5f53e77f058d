// Norms over rows: f16 x, f32 y.
#include "layer_norm_kernels.h"

TERRA_NORM_DEFINE(f16, F16, f32, F32)
