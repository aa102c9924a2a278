// Launch plan of a paged weights call, shared by fa_paged_weights.cu and the translation units that hold
// the kernel instantiations (fa_paged_weights_d*.cu).
#pragma once

#include "fa_paged_weights.cuh"

namespace fa {

struct WeightsPlan {
  CUtensorMap tmQ, tmK;
  PagedWeightsParams params;
  bool half;  // q is fp16 (else bf16)
  bool fp8;
  int grid;
  cudaStream_t stream;
};

int launch_weights_d16(const WeightsPlan& plan);
int launch_weights_d32(const WeightsPlan& plan);
int launch_weights_d64(const WeightsPlan& plan);
int launch_weights_d128(const WeightsPlan& plan);
int launch_weights_d256(const WeightsPlan& plan);

}  // namespace fa
