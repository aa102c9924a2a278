// Instantiations of the paged weights kernel for one head dimension: included with FA_HEAD_DIM defined
// by fa_paged_weights_d*.cu.  q fp16 / bf16, cache of the same type or float8.
#pragma once

#include "fa_paged_launch.h"
#include "fa_paged_weights.cuh"
#include "fa_paged_weights_launch.h"

#ifndef FA_HEAD_DIM
#error "define FA_HEAD_DIM"
#endif

namespace fa {
namespace {

template <typename T, bool FP8, bool ONE>
int launch_weights(const WeightsPlan& plan) {
  using G = WeightsGeo<FA_HEAD_DIM, FP8, ONE>;
  auto kernel = paged_weights_kernel<T, FA_HEAD_DIM, FP8, ONE>;
  static SmemOptIn opt_in;
  if (!opt_in(reinterpret_cast<const void*>(kernel), G::SMEM)) return -7;
  if constexpr (G::SPLIT) {
    static RegsMatch regs_match;
    if (!regs_match(reinterpret_cast<const void*>(kernel), G::REG_LAUNCH)) return -7;
  }
  const int rc = launch_dependent(kernel, dim3(plan.grid), G::THREADS, G::SMEM, plan.stream, plan.tmQ, plan.tmK,
                                  plan.params);
  if (rc != 0 || plan.grid == 1 || plan.params.whole_items) return rc;  // no shared item
  return launch_dependent(paged_weights_join_kernel, dim3(plan.grid - 1), kWeightsBlock, 0, plan.stream,
                          plan.params);
}

int launch_any(const WeightsPlan& plan) {
  if (plan.fp8)
    return plan.half ? launch_weights<__half, true, false>(plan) : launch_weights<__nv_bfloat16, true, false>(plan);
  if (plan.params.whole_items)
    return plan.half ? launch_weights<__half, false, true>(plan) : launch_weights<__nv_bfloat16, false, true>(plan);
  return plan.half ? launch_weights<__half, false, false>(plan) : launch_weights<__nv_bfloat16, false, false>(plan);
}

}  // namespace
}  // namespace fa
