// Paged row kernel for head_dim = 64 (see fa_paged_rows_dispatch.cuh).
#define FA_HEAD_DIM 64
#include "fa_paged_rows_dispatch.cuh"

namespace fa {
int launch_rows_d64(const PagedPlan& plan) { return launch_any(plan); }
}  // namespace fa
