// Paged row kernel for head_dim = 256 (see fa_paged_rows_dispatch.cuh).
#define FA_HEAD_DIM 256
#include "fa_paged_rows_dispatch.cuh"

namespace fa {
int launch_rows_d256(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
