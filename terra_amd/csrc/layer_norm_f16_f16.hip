// Norms over rows: f16 x, f16 y.
#include "layer_norm_kernels.h"

TERRA_NORM_DEFINE(f16, F16, f16, F16)
