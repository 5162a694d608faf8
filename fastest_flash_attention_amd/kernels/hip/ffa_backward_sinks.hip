// The backward kernels of calls with a sliding window and sinks (a unit of its own: they are as
// many again as those without).

#include "ffa_backward_kernels.h"

namespace ffa {

void launch_bwd_sinks(const bwd::BwdParams& p, int dtype, bool softcap, int grid_pre, int grid_dkv,
                      int grid_dq, hipStream_t s) {
  if (dtype == FFA_DTYPE_FP32) {
    launch_f32<true>(p, softcap, grid_pre, s);
  } else if (dtype == FFA_DTYPE_BF16) {
    launch_tag<Sinks<Bf16Tag>>(p, softcap, grid_pre, grid_dkv, grid_dq, s);
  } else {
    launch_tag<Sinks<F16Tag>>(p, softcap, grid_pre, grid_dkv, grid_dq, s);
  }
}

}  // namespace ffa
