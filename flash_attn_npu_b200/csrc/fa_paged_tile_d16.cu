// Paged tile kernel for head_dim = 16 (see fa_paged_tile_dispatch.cuh).
#define FA_HEAD_DIM 16
#include "fa_paged_tile_dispatch.cuh"

namespace fa {
int launch_tile_d16(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
