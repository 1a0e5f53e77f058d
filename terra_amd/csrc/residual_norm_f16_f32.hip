// The end of a half-block for f16 branches and f32 streams.
#include "residual_norm_bwd.h"
#include "residual_norm_fwd.h"

namespace terra {

void tail_fwd_f16_f32(const void* args, bool vec, hipStream_t s) {
  dispatch_fwd<TERRA_DTYPE_F16, TERRA_DTYPE_F32>(*static_cast<const TailArgs*>(args), vec, s);
}

void tail_bwd_f16_f32(const void* args, const TailBwdPlan& plan, bool vec, hipStream_t s) {
  dispatch_bwd<TERRA_DTYPE_F16, TERRA_DTYPE_F32>(*static_cast<const TailArgs*>(args), plan, vec, s);
}

}  // namespace terra
