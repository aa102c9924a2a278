// Launch plan of a paged attention call, shared by the C-ABI front end (fa_paged_api.cu) and the
// translation units that hold the kernel instantiations (fa_paged_rows_d*.cu).
#pragma once

#include <atomic>

#include "fa_paged_attn.cuh"

namespace fa {

// Facts of a kernel that the host needs: rows of a block, keys of a tile, and the boxes of its
// TMA copies.
struct PagedInfo {
  int rows, keys;
  int span;  // bytes of a copied row: the swizzle width
  int cols;  // elements of a copied row
};

struct PagedPlan {
  CUtensorMap tmQ, tmK, tmV;  // tmQ: tile kernel
  PagedAttnParams params;
  bool half;  // q and the output are fp16 (else bf16)
  bool fp8;
  int rows;   // row kernel: rows of a block (8, 16 or 32)
  int grid;
  cudaStream_t stream;
};

int launch_tile_d16(const PagedPlan& plan);
int launch_tile_d32(const PagedPlan& plan);
int launch_tile_d64(const PagedPlan& plan);
int launch_tile_d128(const PagedPlan& plan);
int launch_tile_d256(const PagedPlan& plan);
int launch_rows_d16(const PagedPlan& plan);
int launch_rows_d32(const PagedPlan& plan);
int launch_rows_d64(const PagedPlan& plan);
int launch_rows_d128(const PagedPlan& plan);
int launch_rows_d256(const PagedPlan& plan);

// (Calls of several threads may meet in the two below: what they remember is atomic, and only successes
// are remembered.)

// A kernel's opt-in to more than 48 KB of shared memory, made once per device: the call costs as
// much as a small part of a launch.
struct SmemOptIn {
  std::atomic<bool> done[16] = {};
  bool operator()(const void* kernel, int bytes) {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
    if (dev >= 0 && dev < 16 && done[dev].load(std::memory_order_acquire)) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    if (dev >= 0 && dev < 16) done[dev].store(true, std::memory_order_release);
    return true;
  }
};

// Whether a kernel was built with `regs` registers a thread: setmaxnreg redistributes exactly the launch
// allocation, so a build that differs is refused.
struct RegsMatch {
  std::atomic<bool> known{false};
  bool operator()(const void* kernel, int regs) {
    if (known.load(std::memory_order_relaxed)) return true;
    cudaFuncAttributes attr{};
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    if (attr.numRegs != regs) return false;
    known.store(true, std::memory_order_relaxed);
    return true;
  }
};

// Launch with programmatic dependence on the kernel before it in the stream (see
// wait_for_launch_before): only launch latency and set-up overlap.
template <typename... Params, typename... Args>
int launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, int smem,
                     cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return -7;
}

}  // namespace fa
