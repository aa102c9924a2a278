// Paged tile kernel for head_dim = 32 (see fa_paged_tile_dispatch.cuh).
#define FA_HEAD_DIM 32
#include "fa_paged_tile_dispatch.cuh"

namespace fa {
int launch_tile_d32(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
