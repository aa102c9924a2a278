// Paged row kernel for head_dim = 32 (see fa_paged_rows_dispatch.cuh).
#define FA_HEAD_DIM 32
#include "fa_paged_rows_dispatch.cuh"

namespace fa {
int launch_rows_d32(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
