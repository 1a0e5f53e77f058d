// Norms over rows: bf16 x, f32 y.
#include "layer_norm_kernels.h"

TERRA_NORM_DEFINE(bf16, BF16, f32, F32)
