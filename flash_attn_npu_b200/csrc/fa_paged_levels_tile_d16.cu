// Paged tile kernel of calls behind shared prefixes, head_dim = 16 (see fa_paged_tile_dispatch.cuh).
#define FA_HEAD_DIM 16
#define FA_LEVELS true
#include "fa_paged_tile_dispatch.cuh"

namespace fa {
int launch_levels_tile_d16(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
