// Paged weights kernel for head_dim = 128 (see fa_paged_weights_dispatch.cuh).
#define FA_HEAD_DIM 128
#include "fa_paged_weights_dispatch.cuh"

namespace fa {
int launch_weights_d128(const WeightsPlan& plan) { return launch_any(plan); }
}  // namespace fa
