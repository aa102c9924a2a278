// Paged tile kernel for head_dim = 256 (see fa_paged_tile_dispatch.cuh).
#define FA_HEAD_DIM 256
#include "fa_paged_tile_dispatch.cuh"

namespace fa {
int launch_tile_d256(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
