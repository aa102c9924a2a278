// Instantiations of the paged tile kernel for one head dimension: included with FA_HEAD_DIM defined
// by fa_paged_tile_d*.cu.  q fp16 / bf16, cache of the same type or float8.
#pragma once

#include "fa_paged_launch.h"
#include "fa_paged_tile.cuh"

#ifndef FA_HEAD_DIM
#error "define FA_HEAD_DIM"
#endif

namespace fa {
namespace {

template <typename T, bool FP8>
int launch_tile(const PagedPlan& plan) {
  using G = TileGeo<FA_HEAD_DIM, FP8>;
  auto kernel = paged_tile_kernel<T, FA_HEAD_DIM, FP8>;
  static RegsMatch regs_match;
  if (!regs_match(reinterpret_cast<const void*>(kernel), G::REG_LAUNCH)) return -7;
  static SmemOptIn opt_in;
  if (!opt_in(reinterpret_cast<const void*>(kernel), G::SMEM)) return -7;
  const int rc = launch_dependent(kernel, dim3(plan.grid), G::THREADS, G::SMEM, plan.stream,
                                  plan.tmQ, plan.tmK, plan.tmV, plan.params);
  if (rc != 0) return rc;
  if (plan.grid == 1 || plan.params.whole_items) return 0;  // no shared item
  // a warp to a row: shared items mostly have two or three parts
  constexpr int kRows = 8;
  return launch_dependent(paged_combine_kernel<T, 128, G::TILES, 1, kRows>, dim3(plan.grid - 1, 16),
                          kRows * 32, 0, plan.stream, plan.params);
}

int launch_any(const PagedPlan& plan) {
  if (plan.fp8)
    return plan.half ? launch_tile<__half, true>(plan) : launch_tile<__nv_bfloat16, true>(plan);
  return plan.half ? launch_tile<__half, false>(plan) : launch_tile<__nv_bfloat16, false>(plan);
}

}  // namespace
}  // namespace fa
