// Paged weights kernel for head_dim = 32 (see fa_paged_weights_dispatch.cuh).
#define FA_HEAD_DIM 32
#include "fa_paged_weights_dispatch.cuh"

namespace fa {
int launch_weights_d32(const WeightsPlan& plan) { return launch_any(plan); }
}  // namespace fa
