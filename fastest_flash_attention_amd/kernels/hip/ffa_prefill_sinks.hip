// The prefill kernels of calls with a sliding window and sinks (a unit of its own: they are as
// many again as those without).

#include "ffa_prefill_kernels.h"

namespace ffa {

void launch_sinks(const pf::PrefillParams& p, int dtype, bool softcap, int grid, hipStream_t s) {
  if (dtype == FFA_DTYPE_BF16) {
    launch_tag<Sinks<Bf16Tag>>(p, softcap, grid, s);
  } else if (dtype == FFA_DTYPE_FP16) {
    launch_tag<Sinks<F16Tag>>(p, softcap, grid, s);
  } else {
    launch_f32<true>(p, softcap, grid, s);
  }
}

void launch_split_sinks(const pf::PrefillParams& p, bool bf16, bool softcap, int grid, hipStream_t s) {
  if (bf16) {
    launch_split<Sinks<Bf16Tag>>(p, softcap, grid, s);
  } else {
    launch_split<Sinks<F16Tag>>(p, softcap, grid, s);
  }
}

}  // namespace ffa
