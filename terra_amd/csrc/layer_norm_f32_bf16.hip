// Norms over rows: f32 x, bf16 y.
#include "layer_norm_kernels.h"

TERRA_NORM_DEFINE(f32, F32, bf16, BF16)
