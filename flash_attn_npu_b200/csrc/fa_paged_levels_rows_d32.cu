// Paged row kernel of calls behind shared prefixes, head_dim = 32 (see fa_paged_rows_dispatch.cuh).
#define FA_HEAD_DIM 32
#define FA_LEVELS true
#include "fa_paged_rows_dispatch.cuh"

namespace fa {
int launch_levels_rows_d32(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
