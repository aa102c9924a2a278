// Instantiations of the paged row kernel for one head dimension: included with FA_HEAD_DIM defined
// by fa_paged_rows_d*.cu, so that the head dimensions compile as separate translation units.
//   q fp16 / bf16, cache of the same type or float8, blocks of 8 or 16 rows, or 32 for
//   head_dim <= 128 (with 256 columns there are four warps, which share 16 rows)
#pragma once

#include "fa_paged_launch.h"
#include "fa_paged_rows.cuh"

#ifndef FA_HEAD_DIM
#error "define FA_HEAD_DIM"
#endif

namespace fa {
namespace {

template <typename T, bool FP8, int ROWS>
int launch_rows(const PagedPlan& plan) {
  using G = RowsGeo<FA_HEAD_DIM, FP8, ROWS>;
  auto kernel = paged_rows_kernel<T, FA_HEAD_DIM, FP8, ROWS>;
  if constexpr (G::SPLIT) {
    static RegsMatch regs_match;
    if (!regs_match(reinterpret_cast<const void*>(kernel), G::REG_LAUNCH)) return -7;
  }
  static SmemOptIn opt_in;
  if (!opt_in(reinterpret_cast<const void*>(kernel), G::SMEM)) return -7;
  const int rc = launch_dependent(kernel, dim3(plan.grid), G::THREADS, G::SMEM, plan.stream,
                                  plan.tmK, plan.tmV, plan.params);
  if (rc != 0) return rc;
  if (plan.grid == 1 || plan.params.whole_items) return 0;  // no shared item
  const int64_t most = static_cast<int64_t>(plan.params.seqs.total) * plan.params.group;
  const unsigned rows = static_cast<unsigned>(most < G::ROWS ? most : G::ROWS);
  constexpr int kWarps = 4;
  return launch_dependent(paged_combine_kernel<T, G::ROWS, 1, kWarps, 1>, dim3(plan.grid - 1, rows),
                          kWarps * 32, 0, plan.stream, plan.params);
}

template <typename T, bool FP8>
int launch_blocks(const PagedPlan& plan) {
  if (plan.rows == 8) return launch_rows<T, FP8, 8>(plan);
  if constexpr (FA_HEAD_DIM <= 128) {
    if (plan.rows == 32) return launch_rows<T, FP8, 32>(plan);
  }
  return launch_rows<T, FP8, 16>(plan);
}

int launch_any(const PagedPlan& plan) {
  if (plan.fp8)
    return plan.half ? launch_blocks<__half, true>(plan) : launch_blocks<__nv_bfloat16, true>(plan);
  return plan.half ? launch_blocks<__half, false>(plan) : launch_blocks<__nv_bfloat16, false>(plan);
}

}  // namespace
}  // namespace fa
