// Paged weights kernel for head_dim = 256 (see fa_paged_weights_dispatch.cuh).
#define FA_HEAD_DIM 256
#include "fa_paged_weights_dispatch.cuh"

namespace fa {
int launch_weights_d256(const WeightsPlan& plan) { return launch_any(plan); }
}  // namespace fa
