// Paged weights kernel for head_dim = 16 (see fa_paged_weights_dispatch.cuh).
#define FA_HEAD_DIM 16
#include "fa_paged_weights_dispatch.cuh"

namespace fa {
int launch_weights_d16(const WeightsPlan& plan) { return launch_any(plan); }
}  // namespace fa
