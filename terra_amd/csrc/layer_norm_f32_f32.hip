// Norms over rows: f32 x, f32 y.
#include "layer_norm_kernels.h"

TERRA_NORM_DEFINE(f32, F32, f32, F32)
