// Paged row kernel of calls behind shared prefixes, head_dim = 256 (see fa_paged_rows_dispatch.cuh).
#define FA_HEAD_DIM 256
#define FA_LEVELS true
#include "fa_paged_rows_dispatch.cuh"

namespace fa {
int launch_levels_rows_d256(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
