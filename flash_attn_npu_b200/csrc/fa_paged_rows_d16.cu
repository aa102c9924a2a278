// Paged row kernel for head_dim = 16 (see fa_paged_rows_dispatch.cuh).
#define FA_HEAD_DIM 16
#include "fa_paged_rows_dispatch.cuh"

namespace fa {
int launch_rows_d16(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
