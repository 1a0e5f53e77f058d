// Norms over rows: bf16 x, bf16 y.
#include "layer_norm_kernels.h"

TERRA_NORM_DEFINE(bf16, BF16, bf16, BF16)
